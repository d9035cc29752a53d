"""``MoELM`` and ``ExpertAdamW``: a training program around the MoE layer, from token ids to the updated weights.

The reference ends at the layer; what its users write around it (an embedding, the loss over the vocabulary, clipping, the
optimizer) is here in its smallest form, on the library's own operators: ``linear_cross_entropy`` for the output
projection and the loss, ``grad_norm`` over replicated and expert weights, ``adamw_step_`` with the clipping in it; and with ``mixer``
and ``train_router`` a block around the experts: ``layer_norm`` with the residual stream, ``gated_scan`` along the sequences,
``balanced_router``.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import nn

from ..buffer import Buffer
from ..ops.linear_loss import linear_cross_entropy
from ..ops.norm import layer_norm
from ..ops.recurrence import gated_scan, gated_scan_step_
from ..ops.tensor_lists import adamw_step_, grad_norm
from .moe_layer import StreamMoE


class Mixer(nn.Module):
    """Mixes the tokens of a sequence: a projection to values and gates, :func:`gated_scan`, a projection back; with the norms in front of it and
    behind it (in front of the experts)."""

    def __init__(self, hidden: int, generator: torch.Generator, device=None):
        super().__init__()
        weight = lambda *shape: nn.Parameter((torch.randn(*shape, generator=generator) / math.sqrt(hidden)).to(torch.bfloat16).to(device))
        plain = lambda value: nn.Parameter(torch.full((hidden,), value, dtype=torch.bfloat16, device=device))
        self.w_in, self.w_out = weight(2 * hidden, hidden), weight(hidden, hidden)
        # channels that forget soon beside channels that remember for hundreds of tokens
        self.gate_bias = nn.Parameter(torch.linspace(0.0, 6.0, hidden).to(torch.bfloat16).to(device))
        self.norm_weight, self.norm_bias = plain(1.0), plain(0.0)
        self.expert_norm_weight, self.expert_norm_bias = plain(1.0), plain(0.0)

    def values_and_gates(self, x: torch.Tensor):
        values, gates = torch.nn.functional.linear(x, self.w_in).chunk(2, dim=-1)
        return values, gates + self.gate_bias


class MoELM(nn.Module):
    """Embedding, ``num_layers`` residual MoE layers on normalised rows, output projection.

    Without ``mixer`` there is no token mixer: it models the next token from the present one, which is what a training step needs to be
    exercised.  With it each layer is a :class:`Mixer` and the experts, ``tokens`` are ``[B, T]``, or packed sequences ``[N]`` with
    ``offsets`` (see :func:`gated_scan`), and :meth:`step` goes on token by token.

    ``train_router``: the gates are trained; ``forward`` adds their balance and z losses, times ``balance_coef`` and ``z_coef``, to a mean
    loss that is differentiated."""

    def __init__(self, vocab: int, hidden: int, ffn: int, num_experts: int, top_k: int, num_layers: int, buffer: Buffer, *,
                 device=None, seed: int = 0, mixer: bool = False, train_router: bool = False, balance_coef: float = 0.01, z_coef: float = 0.001):
        super().__init__()
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.embedding = nn.Parameter(torch.randn(vocab, hidden, generator=g).to(torch.bfloat16).to(device))
        self.head = nn.Parameter((torch.randn(vocab, hidden, generator=g) * 0.02).to(torch.bfloat16).to(device))
        self.layers = nn.ModuleList(StreamMoE(hidden, ffn, num_experts, top_k, buffer, device=device, seed=seed + i, train_router=train_router)
                                    for i in range(num_layers))
        self.mixers = nn.ModuleList(Mixer(hidden, g, device) for _ in range(num_layers if mixer else 0))
        self.hidden, self.train_router, self.balance_coef, self.z_coef = hidden, train_router, balance_coef, z_coef
        self.buffer = buffer

    def hidden_states(self, tokens: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        for layer in self.layers:        # (a forward whose losses nobody took has left its graph with them: it must be gone before this one meets the same
            layer.last_route = None      # parameters, which a captured forward could not share with it)
        x = torch.nn.functional.embedding(tokens.reshape(-1), self.embedding)
        counts = None            # (rows of a packed batch that belong to no sequence are padding, and none of the gates' business)
        if offsets is not None and self.train_router and torch.is_grad_enabled():
            row = torch.arange(x.shape[0], device=x.device)
            counts = (row >= offsets[0]) & (row < offsets[-1])
        if not self.mixers:
            for layer in self.layers:
                x = x + layer(torch.nn.functional.rms_norm(x, x.shape[-1:]), counts)
            return torch.nn.functional.rms_norm(x, x.shape[-1:])
        shape = x.shape if offsets is not None else (*tokens.shape, self.hidden)
        mix = lambda i, values, gates: gated_scan(values.view(shape), gates.view(shape), offsets=offsets, buffer=self.buffer).view(x.shape)
        return self._blocks(x, mix, counts)

    def _blocks(self, x: torch.Tensor, mix, counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The layers with their mixers; ``mix(i, values, gates)`` is what runs along the sequences, ``counts`` the tokens that the gates' losses take."""
        added = None
        for i, (mixer, layer) in enumerate(zip(self.mixers, self.layers)):
            if added is None:
                y = layer_norm(x, mixer.norm_weight, mixer.norm_bias)
            else:
                y, x = layer_norm(added, mixer.norm_weight, mixer.norm_bias, residual=x)
            mixed = torch.nn.functional.linear(mix(i, *mixer.values_and_gates(y)), mixer.w_out)
            y, x = layer_norm(mixed, mixer.expert_norm_weight, mixer.expert_norm_bias, residual=x)
            added = layer(y, counts)
        return layer_norm(added, residual=x)[0]

    def router_losses(self) -> torch.Tensor:
        """The gates' losses of the last forward, with their coefficients, averaged over the layers; once, as :meth:`StreamMoE.router_losses`."""
        losses = [layer.router_losses() for layer in self.layers]
        return sum(self.balance_coef * balance + self.z_coef * z for balance, z in losses) / len(losses)

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor, reduction: str = "mean", offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        loss = linear_cross_entropy(self.hidden_states(tokens, offsets), self.head, targets.reshape(-1), reduction=reduction, buffer=self.buffer)
        if self.train_router and reduction == "mean" and torch.is_grad_enabled():
            loss = loss + self.router_losses()
        return loss

    @torch.no_grad()
    def log_probs(self, tokens: torch.Tensor, targets: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """log P(target) of every token, shaped like ``tokens``."""
        return -self.forward(tokens, targets, reduction="none", offsets=offsets).view(tokens.shape)

    def states(self, sequences: int) -> List[torch.Tensor]:
        """What :meth:`step` keeps of ``sequences`` sequences, before their first token."""
        return [torch.zeros(sequences, self.hidden, device=self.head.device) for _ in self.mixers]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, states: List[torch.Tensor]) -> torch.Tensor:
        """One more token ``[S]`` of every sequence: the next token's logits ``[S, V]``; ``states`` go on in place.  For a model with mixers."""
        if not self.mixers:
            raise RuntimeError("step() continues the states of a model with mixers: MoELM(mixer=True)")
        x = torch.nn.functional.embedding(tokens, self.embedding)
        x = self._blocks(x, lambda i, values, gates: gated_scan_step_(states[i], values, gates))
        return torch.nn.functional.linear(x, self.head)

    def replicated_parameters(self) -> List[nn.Parameter]:
        gates = [layer.w_gate for layer in self.layers] if self.train_router else []
        return [self.embedding, self.head] + gates + [p for mixer in self.mixers for p in mixer.parameters()]

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
