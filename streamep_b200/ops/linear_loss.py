"""The output projection with softmax cross entropy (``csrc/linear_loss_kernels.cu``), without logits in memory.

No counterpart in the reference, which ends at the MoE layer: its users compute the loss with PyTorch, logits of
``[tokens, vocabulary]`` and all.
"""
from __future__ import annotations

import torch

from .grouped_gemm import _rt

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", buffer=None) -> torch.Tensor:
    """``cross_entropy(x @ weight.T, targets)`` for hidden states ``x [..., H]`` and an output projection
    ``weight [V, H]`` (both bf16; logits, statistics and losses in fp32), differentiable in both.

    The gradients are bf16.  Their sums are fp32, over terms ``dz * weight`` and ``dz * x`` whose ``dz``, the gradient of a
    logit, is rounded to bf16 first (calls of up to 64 tokens keep 16 bits of it): an element is off by at most
    2^-8 of the sum of its terms' magnitudes and 2^-8 of itself, 2e-3 of a gradient in 2-norm where terms do not cancel.
    Elements of ``x`` that are not finite make ``weight``'s gradient NaN, those of ignored tokens too (zero times infinity).

    Neither pass keeps logits: the forward reduces each 256 x 256 tile of them to softmax statistics in the epilogue
    of the product, the backward computes them again piece by piece of the vocabulary (workspace: two buffers of at
    most about 256 MB, and fp32 sums of ``x``'s gradient; the forward's statistics take 8 bytes for every token and 128
    columns).  A repeated call gives the same bits.  Rows that lie a multiple of 128 bytes apart (``H``, or the stride of a padded
    matrix's ``[:, :H]``, a multiple of 64) are read 13 to 40 % faster than others.

    ``targets [...]`` int64; tokens whose target is ``ignore_index`` have no loss, count for nothing in the mean and
    get zero gradients.  ``reduction``: ``"mean"`` over the counted tokens (NaN without any, gradients zero),
    ``"sum"``, or ``"none"`` for a loss per token (float32, shaped like ``targets``).  A target outside the
    vocabulary makes the loss and the gradients NaN and is reported, like a wait on the device that gave up, by
    ``buffer.check_status()``, or without ``buffer`` by ``streamep_b200.ops.check_status()``.

    Under ``torch.no_grad()`` only the forward runs: ``-linear_cross_entropy(..., reduction="none")`` are the
    log-probabilities of given tokens, for one token as for a batch.  There is no second derivative.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)} (got {reduction!r})")
    if x.dim() < 1 or x.shape[:-1] != targets.shape:
        raise ValueError(f"targets must have the shape of x without its last dimension (x {tuple(x.shape)}, targets {tuple(targets.shape)})")
    if not x.is_cuda:
        raise ValueError(f"x must be a [..., H] bf16 CUDA tensor (got one on {x.device})")
    loss = _rt(buffer, x.device).linear_loss(x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x, weight, targets.reshape(-1),
                                             int(ignore_index), _REDUCTIONS[reduction])
    return loss.view(targets.shape) if reduction == "none" else loss
