"""The router with what its training needs (``csrc/route_kernels.cu``): the experts' counts, a balance and a z loss, gradients.

No counterpart in the reference, which has no router.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .grouped_gemm import _rt


class BalancedRoute(NamedTuple):
    """What :func:`balanced_router` returns."""

    topk_idx: torch.Tensor             # [T, K] int64
    topk_weights: torch.Tensor         # [T, K] float32, differentiable
    is_token_in_rank: torch.Tensor     # [T, num_ranks] bool
    balance_loss: torch.Tensor         # 0-dim float32, differentiable
    z_loss: torch.Tensor               # 0-dim float32, differentiable
    expert_counts: torch.Tensor        # [E] int64


def balanced_router(x: torch.Tensor, w_gate: torch.Tensor, top_k: int, num_ranks: int = 1, renormalize: bool = True, *,
                    mask: Optional[torch.Tensor] = None, buffer=None) -> BalancedRoute:
    """:func:`router_topk` as a differentiable function of ``x [T, H]`` and ``w_gate [E, H]`` (both bf16), with the losses that keep its
    experts in use::

        p = softmax(x @ w_gate.T);   topk_idx, topk_weights: the top_k largest of each row, divided by their sum with ``renormalize``
        expert_counts[e] = tokens that chose e
        balance_loss = E * sum_e expert_counts[e] / (top_k * n) * mean_t p[t, e]          # 1 where all experts are used alike
        z_loss = mean_t logsumexp(x @ w_gate.T)[t] ** 2

    ``mask [T]`` (bool): tokens that count; the others (padding) are routed all the same, but are left out of counts, means and
    ``n`` (both losses are 0 without any that counts).  Whatever they hold, losses and the losses' gradient of ``x`` are the same; but the gradient of
    ``w_gate`` multiplies their ``x`` with zero, which an infinity or NaN survives.  Every rank's losses are those of its own tokens.

    The choice itself and the counts have no gradient; weights and losses do, for ``x`` and ``w_gate`` (bf16), by ``dz @ w_gate`` and
    ``dz.T @ x``.  The gradient ``dz`` of the logits is formed in 32 bits; the products take it as the sum of two bf16 numbers (2^-16 of it) up
    to 128 experts, and above as one (2^-8 of it, as a bf16 logit's gradient would be): in 2-norm the gradients are then 2.3e-3 off instead of the 1.7e-3 that is the
    rounding of the results.  Sums are in 32 bits.  There is no second derivative.  A repeated call gives the same bits.  Ties go to the lowest expert.  1 to 512 experts, up to 32 of them a token, ``H`` a multiple of 8.

    A wait on the device that gave up is reported by ``buffer.check_status()``, or without ``buffer`` by
    ``streamep_b200.ops.check_status()``."""
    if not x.is_cuda:
        raise ValueError(f"x must be a [T, H] bf16 CUDA tensor (got one on {x.device})")
    return BalancedRoute(*_rt(buffer, x.device).balanced_router(x, w_gate, int(top_k), int(num_ranks), bool(renormalize), mask))
