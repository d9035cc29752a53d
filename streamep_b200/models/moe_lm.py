"""``MoELM`` and ``ExpertAdamW``: a training program around the MoE layer, from token ids to the updated weights.

The reference ends at the layer; what its users write around it (an embedding, the loss over the vocabulary, clipping, the
optimizer) is here in its smallest form, on the library's own operators: ``linear_cross_entropy`` for the output
projection and the loss, ``grad_norm`` over replicated and expert weights, ``adamw_step_`` with the clipping in it.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import nn

from ..buffer import Buffer
from ..ops.linear_loss import linear_cross_entropy
from ..ops.tensor_lists import adamw_step_, grad_norm
from .moe_layer import StreamMoE


class MoELM(nn.Module):
    """Embedding, ``num_layers`` residual MoE layers on RMS-normalised rows, output projection.  There is no token mixer:
    it models the next token from the present one, which is what a training step needs to be exercised."""

    def __init__(self, vocab: int, hidden: int, ffn: int, num_experts: int, top_k: int, num_layers: int, buffer: Buffer, *,
                 device=None, seed: int = 0):
        super().__init__()
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.embedding = nn.Parameter(torch.randn(vocab, hidden, generator=g).to(torch.bfloat16).to(device))
        self.head = nn.Parameter((torch.randn(vocab, hidden, generator=g) * 0.02).to(torch.bfloat16).to(device))
        self.layers = nn.ModuleList(StreamMoE(hidden, ffn, num_experts, top_k, buffer, device=device, seed=seed + i)
                                    for i in range(num_layers))
        self.buffer = buffer

    def hidden_states(self, tokens: torch.Tensor) -> torch.Tensor:
        x = torch.nn.functional.embedding(tokens.reshape(-1), self.embedding)
        for layer in self.layers:
            x = x + layer(torch.nn.functional.rms_norm(x, x.shape[-1:]))
        return torch.nn.functional.rms_norm(x, x.shape[-1:])

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor, reduction: str = "mean") -> torch.Tensor:
        return linear_cross_entropy(self.hidden_states(tokens), self.head, targets.reshape(-1), reduction=reduction, buffer=self.buffer)

    @torch.no_grad()
    def log_probs(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """log P(target) of every token, shaped like ``tokens``."""
        return -self.forward(tokens, targets, reduction="none").view(tokens.shape)

    def replicated_parameters(self) -> List[nn.Parameter]:
        return [self.embedding, self.head]

    def expert_parameters(self) -> List[nn.Parameter]:
        return [p for layer in self.layers for p in (layer.w1, layer.w2)]


class ExpertAdamW:
    """AdamW with float32 master copies for a model whose expert weights are sharded over ``group`` and whose other
    weights are replicated.  ``step()`` takes the norm over everything (each expert counted once), clips and updates: one pass
    over the gradients for the norm, one over all state.  With several ranks it first averages the replicated gradients over
    the group and divides the experts' by its size, in place: an all-reduce and a division a tensor, one more pass over the
    gradients.  The all-reduces are collective: a replicated parameter has a gradient on every rank or on none."""

    def __init__(self, replicated, experts, *, lr: float, betas=(0.9, 0.95), eps: float = 1e-8, weight_decay: float = 0.1,
                 max_norm: Optional[float] = 1.0, skip_nonfinite: bool = True, group=None):
        self.replicated, self.experts, self.group = list(replicated), list(experts), group
        self.params = self.replicated + self.experts
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.max_norm, self.skip_nonfinite = max_norm, skip_nonfinite
        self.masters = [p.detach().to(torch.float32, copy=True) for p in self.params]      # (of float32 parameters too: both are written)
        self.exp_avgs = [torch.zeros_like(m) for m in self.masters]
        self.exp_avg_sqs = [torch.zeros_like(m) for m in self.masters]
        # updates made, of each parameter: a skipped one is none, nor one without a gradient.  Parameters that have taken part in the same
        # updates share one number, and an update.
        start = torch.zeros((), dtype=torch.int64, device=self.masters[0].device if self.masters else None)
        self.steps = [start] * len(self.params)

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    @torch.no_grad()
    def step(self) -> torch.Tensor:
        """Returns the norm (0-dim, on the device).  Parameters without a gradient are left out: their moments and their count of
        updates stay."""
        ranks = self.group.size() if self.group is not None else 1
        if ranks > 1:
            # a mean over the ranks' tokens: experts already hold the sum of what all ranks sent them
            for p in self.replicated:
                if p.grad is not None:
                    torch.distributed.all_reduce(p.grad, group=self.group)
            for p in self.params:
                if p.grad is not None:
                    p.grad.div_(ranks)
        live = [i for i, p in enumerate(self.params) if p.grad is not None]
        grads = [self.params[i].grad for i in live]
        sharded = [self.params[i].grad for i in live if i >= len(self.replicated)] if ranks > 1 else []
        norm = grad_norm(grads[:len(grads) - len(sharded)], sharded=sharded, group=self.group)
        made = norm < math.inf if self.skip_nonfinite else 1
        for together in self._same_steps(live):
            step = self.steps[together[0]]
            step += made
            pick = lambda tensors: [tensors[i] for i in together]
            adamw_step_(pick(self.params), [self.params[i].grad for i in together], pick(self.exp_avgs), pick(self.exp_avg_sqs),
                        masters=pick(self.masters), step=step, lr=self.lr, betas=self.betas, eps=self.eps,
                        weight_decay=self.weight_decay, norm=norm, max_norm=self.max_norm, skip_nonfinite=self.skip_nonfinite)
        return norm

    def _same_steps(self, live: List[int]) -> List[List[int]]:
        """``live`` by their counts; one that others hold as well, who are not in ``live``, is copied first."""
        groups = {}
        for i in live:
            groups.setdefault(id(self.steps[i]), []).append(i)
        if len(live) < len(self.params):
            left = {id(self.steps[i]) for i in set(range(len(self.params))).difference(live)}
            for key, members in groups.items():
                if key in left:
                    own = self.steps[members[0]].clone()
                    for i in members:
                        self.steps[i] = own
        return list(groups.values())

    def state_dict(self) -> dict:
        steps = torch.stack(self.steps) if self.steps else torch.zeros(0, dtype=torch.int64)
        return {"steps": steps, "masters": self.masters, "exp_avgs": self.exp_avgs, "exp_avg_sqs": self.exp_avg_sqs}

    @torch.no_grad()
    def load_state_dict(self, state: dict) -> None:
        numbers = torch.as_tensor(state["steps"]).expand(len(self.params)).tolist()        # (one for all of them will do)
        shared = {n: torch.tensor(n, dtype=torch.int64, device=self.masters[0].device) for n in set(numbers)}
        self.steps = [shared[n] for n in numbers]
        for name in ("masters", "exp_avgs", "exp_avg_sqs"):
            for mine, theirs in zip(getattr(self, name), state[name], strict=True):
                mine.copy_(theirs)
        for p, m in zip(self.params, self.masters):
            p.copy_(m)
