"""A gated linear recurrence along sequences (``csrc/scan_kernels.cu``), and its form for one more token.

No counterpart in the reference, which ends at the MoE layer.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ext
from .grouped_gemm import _rt


def gated_scan(x: torch.Tensor, gate: torch.Tensor, *, initial_state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
               return_state: bool = False, buffer=None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``h_t = sigmoid(gate_t) * h_{t-1} + (1 - sigmoid(gate_t)) * x_t`` along every sequence, channel by channel.

    ``x`` and ``gate`` (the gate before its sigmoid) are both bf16 or both float32: ``[B, T, D]``, or packed sequences ``[N, D]`` whose
    first rows ``offsets [S + 1]`` (int32 or int64, on the device) holds, sequence ``s`` being rows ``offsets[s]`` to
    ``offsets[s + 1]``.  Sequences may be empty.  Rows before the first and behind the last one are not read; ``h`` and the gradients
    are zero there.  Views with gaps between rows (the halves of one projection's output) are read in place.

    Returns ``h`` like ``x``; with ``return_state`` ``(h, final_state)``, float32 ``[S, D]``: the unrounded state behind each sequence's last
    row, which continues it as another call's ``initial_state`` (float32, zeros without one).  An empty sequence hands its state on.

    Differentiable in ``x``, ``gate`` and ``initial_state``; there is no second derivative.  The state and its gradient are carried in 32 bits (a state
    that lasts for many rows follows its inputs without drift: what a row keeps and takes adds up to 1).  The gate's gradient
    ``g_t * s (1 - s) * (h_{t-1} - x_t)`` takes ``h_{t-1}`` as it was returned, rounded to the type of ``x``.  A repeated call gives the
    same bits.  An infinity or NaN stays within its sequence and channel.

    Offsets that decrease or point outside leave the sequences that they belong to undefined, and are reported, like a wait on the device that gave
    up, by ``buffer.check_status()``, or without ``buffer`` by ``streamep_b200.ops.check_status()``."""
    if not x.is_cuda:
        raise ValueError(f"x must be a bf16 or float32 CUDA tensor (got one on {x.device})")
    out = _rt(buffer, x.device).gated_scan(x, gate, initial_state, offsets, return_state)
    return (out[0], out[1]) if return_state else out[0]


def gated_scan_step_(state: torch.Tensor, x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    """One more token for every sequence: ``state [S, D]`` (float32) becomes ``sigmoid(gate) * state + (1 - sigmoid(gate)) * x`` in
    place, for ``x`` and ``gate [S, D]`` (both bf16 or both float32); returns the new state in the type of ``x``.  No gradient."""
    return _ext.load().gated_scan_step(state, x, gate)
