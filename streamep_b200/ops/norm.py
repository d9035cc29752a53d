"""Normalisation of rows (``csrc/norm_kernels.cu``), with the residual stream added on the way.

No counterpart in the reference, which ends at the MoE layer.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ext


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Rows of ``x [..., H]`` (bf16 or float32) with mean 0 and variance 1, scaled and shifted::

        y = (x - mean) / sqrt(var + eps) * weight + bias

    ``weight`` and ``bias [H]`` are bf16 or float32, whatever ``x`` is, and may be left out.  With ``residual`` (like ``x``) the rows are
    ``x + residual``, and the call returns ``(y, sum)``: the sum, rounded to the type of ``x``, is the residual stream from here on.
    ``y`` comes from the sum before its rounding.

    Differentiable in all four tensors; there is no second derivative.  Mean and variance (of centred values), and all sums, are
    formed in 32 bits, the gradients of ``x + residual`` before its rounding too (so both are kept for the backward, not the sum).  A
    repeated call gives the same bits.  A row with an infinity or NaN becomes NaN, and so do weight and bias' gradients that it has a part in; squares above the
    range of 32 bits (values 1.8e19 from the mean) make a row's outputs 0."""
    out = _ext.load().norm_rows(x, weight, bias, residual, True, float(eps))
    return (out[0], out[1]) if residual is not None else out[0]


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``x / sqrt(mean(x * x) + eps) * weight``: as :func:`layer_norm`, without mean and bias."""
    out = _ext.load().norm_rows(x, weight, None, residual, False, float(eps))
    return (out[0], out[1]) if residual is not None else out[0]
