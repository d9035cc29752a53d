"""Operators over lists of tensors (``csrc/list_kernels.cu``): the norm of all gradients, clipping, and AdamW.

No counterpart in the reference, which ends at the MoE layer.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _ext


def _over_ranks(group) -> bool:
    return group is not None and group.size() > 1


def _total(grads, sharded, group):
    """The norm, with the sharded gradients' squares summed over the ranks of ``group`` (every rank takes part, also one
    that holds no sharded gradient)."""
    C = _ext.load()
    if not _over_ranks(group):
        return C.list_norm(grads + sharded)[0]
    # (an empty list beside one with tensors: on their device, whichever is current)
    squares = C.list_norm(grads)[1] if grads or not sharded else None
    parts = C.list_norm(sharded)[1] if sharded or not grads else torch.zeros_like(squares)
    if squares is None:
        squares = torch.zeros_like(parts)
    torch.distributed.all_reduce(parts, group=group)
    return (squares + parts).sqrt().float()


def grad_norm(grads: Sequence[torch.Tensor], *, sharded: Sequence[torch.Tensor] = (), group=None) -> torch.Tensor:
    """The 2-norm of all elements of ``grads`` (bf16 or float32, any mix, on one device), a 0-dim float32 tensor on the
    device; nothing is read on the host.

    ``sharded``: gradients of which every rank of ``group`` holds others (the experts' weights under expert
    parallelism); their squares are summed over the group, those of ``grads`` (the same on all ranks) are counted
    once.  With a ``group`` of several ranks the call is collective.  Squares are formed in 32 bits: elements above 1.8e19 give an infinite norm."""
    return _total(list(grads), list(sharded), group)


def clip_grad_norm_(grads: Sequence[torch.Tensor], max_norm: float, *, sharded: Sequence[torch.Tensor] = (), group=None) -> torch.Tensor:
    """Scales all gradients in place by ``min(1, max_norm / (norm + 1e-6))`` and returns their norm before that (see
    :func:`grad_norm`).  Below the limit the gradients are read once and not written (those with gaps in memory, which go through
    copies, are written back as they were).  A norm of NaN makes all
    gradients NaN, an infinite one makes them 0 (and NaN where they are infinite), as ``torch.nn.utils`` has it.
    Tensors that share memory are refused (strided views, which go through copies, are not compared), and so are expanded ones.

    Where an update follows, :func:`adamw_step_` applies the same factor on its way and no pass over the gradients is
    needed for it."""
    grads, sharded = list(grads), list(sharded)
    C = _ext.load()
    if not _over_ranks(group):
        return C.list_clip(grads + sharded, float(max_norm))
    norm = _total(grads, sharded, group)
    C.list_scale(grads + sharded, norm, float(max_norm))
    return norm


def adamw_step_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                exp_avg_sqs: Sequence[torch.Tensor], *, step: Union[int, torch.Tensor], lr: float, betas: Tuple[float, float] = (0.9, 0.999),
                eps: float = 1e-8, weight_decay: float = 0.0, masters: Optional[Sequence[torch.Tensor]] = None,
                norm: Optional[torch.Tensor] = None, max_norm: Optional[float] = None, skip_nonfinite: bool = False) -> None:
    """One AdamW step (decoupled weight decay) on all of ``params`` in place, in one launch per 512 tensors::

        g = grad * min(1, max_norm / (norm + 1e-6))        # norm: grad_norm(grads); without max_norm g = grad
        exp_avg = b1 * exp_avg + (1 - b1) * g;  exp_avg_sq = b2 * exp_avg_sq + (1 - b2) * g * g
        w = w * (1 - lr * weight_decay) - lr * (exp_avg / (1 - b1**step)) / (sqrt(exp_avg_sq / (1 - b2**step)) + eps)

    Parameters and gradients are bf16 or float32, the moments float32, all arithmetic 32 bits.  With ``masters``
    (float32) ``w`` is the master copy and the parameter becomes its rounding.

    ``step``, the number of this update, counts from 1.  Like ``lr`` it may be a number of the host, which a captured graph
    repeats; or one int64 number on the parameters' device, read when the update runs (below 1 the weights become NaN).
    ``skip_nonfinite``: leave everything as it is when ``norm`` is not finite, decided on the device.  An update that was
    skipped must not be counted: ``steps += norm < math.inf`` before the call, and ``step=steps``, does that without reading
    the norm on the host."""
    if max_norm is not None and norm is None:
        raise ValueError("max_norm needs the gradients' norm (grad_norm)")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative (got {max_norm})")
    if skip_nonfinite and norm is None:
        raise ValueError("skip_nonfinite needs the gradients' norm (grad_norm)")
    if masters is not None and len(masters) != len(params):
        raise ValueError(f"{len(params)} params and {len(masters)} masters")
    device_step = step if isinstance(step, torch.Tensor) else None
    _ext.load().list_adamw(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), list(masters) if masters is not None else [], norm,
                           0 if device_step is not None else int(step), device_step, float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                           -1.0 if max_norm is None else float(max_norm), bool(skip_nonfinite))
