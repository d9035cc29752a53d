"""A block around the experts, measured: the normalisation in front of a layer, a gated linear recurrence that mixes the
tokens of a sequence, and routing that is trained (balance loss, counts, the gate's gradients).

Four kinds of call, each through the public entry points:

* ``norm``   ``layer_norm``: rows normalised to mean 0 and variance 1, scaled and shifted, after adding the residual stream where
             there is one; with ``train`` the gradients of rows, weight and bias
* ``scan``   ``gated_scan``: ``h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t`` along every sequence, dense or packed;
             with ``train`` the gradients of ``x``, ``gate`` and the initial state
* ``step``   ``gated_scan_step_``: one more token for each sequence, the state updated in place
* ``route``  ``balanced_router``: gate, softmax, top-k, weights, ranks, the experts' counts, balance and z loss; with ``train`` the
             gradients of the hidden states and of the gate's weight

Where ``own`` is false the same is computed in its plain form: 32-bit tensors, one elementary operation after another.
"""
import math
import random

import torch

own = False

#: Upper ends of the ranges that ``draw`` samples.
MAX_ROWS, MAX_HIDDEN, MAX_LENGTH, MAX_CHANNELS, MAX_SEQUENCES, MAX_EXPERTS, MAX_TOPK = 65536, 8192, 131072, 4096, 512, 512, 8
EPS = 1e-5
#: Candidates whose first top_k + 1 logits come closer than this are not taken as tokens: their order would be a matter of rounding.
GAP = 3e-4


def listed():
    return [
        # The benchmark's default layer: the residual stream joined by a layer's output, normalised for the next one.
        dict(name="norm training", kind="norm", rows=8192, hidden=2048, dtype="bf16", weights="bf16", residual=True, bias=True, train=True),
        # The benchmark's widest rows, a long batch.
        dict(name="norm wide", kind="norm", rows=32768, hidden=7168, dtype="bf16", weights="fp32", residual=True, bias=True, train=True),
        # Odd rows in 32 bits: no row but the first starts on a 16-byte boundary.
        dict(name="norm odd", kind="norm", rows=1777, hidden=1001, dtype="fp32", weights="fp32", residual=False, bias=True, train=True),
        # One token of a decoding step: latency.
        dict(name="norm one token", kind="norm", rows=1, hidden=4096, dtype="bf16", weights="bf16", residual=True, bias=False, train=False),
        # The default layer's tokens as four sequences, x and gate as halves of one projection's output.
        dict(name="scan training", kind="scan", sequences=4, tokens=8192, packed=False, channels=2048, dtype="bf16", joint=True, state=False, train=True),
        # One long document.
        dict(name="scan long", kind="scan", sequences=1, tokens=131072, packed=False, channels=1024, dtype="bf16", joint=False, state=False, train=True),
        # Packed documents of every length (empty ones and single tokens among them), continued from a state, channels no multiple
        # of a vector, rows behind the last document.
        dict(name="scan packed", kind="scan", sequences=9, tokens=7457, packed=True, channels=1001, dtype="fp32", joint=False,
             state=True, train=True),
        # One more token for each of 64 sequences.
        dict(name="step", kind="step", sequences=64, channels=2048, dtype="bf16"),
        # The default layer's routing over the experts of eight ranks.
        dict(name="route training", kind="route", tokens=8192, hidden=2048, experts=64, top_k=6, ranks=8, renormalize=True, masked=0.0, train=True),
        # The benchmark's skewed configuration: wide rows, many experts, a quarter of the batch is padding.
        dict(name="route many experts", kind="route", tokens=16384, hidden=7168, experts=256, top_k=8, ranks=8, renormalize=True, masked=0.25,
             train=True),
        # Ragged sizes, probabilities as weights.
        dict(name="route ragged", kind="route", tokens=1777, hidden=1000, experts=60, top_k=3, ranks=4, renormalize=False, masked=0.1, train=True),
        # A decoding step's routing with its counts.
        dict(name="route decoding", kind="route", tokens=64, hidden=4096, experts=256, top_k=8, ranks=1, renormalize=True, masked=0.0, train=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(["norm", "scan", "step", "route"], [3, 3, 1, 3])[0]
    if kind == "norm":
        step = rng.choice([64, 8, 1])
        hidden = max(step, _log_int(rng, 8, MAX_HIDDEN) // step * step)
        return dict(kind=kind, rows=_log_int(rng, 1, MAX_ROWS), hidden=hidden, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    weights=rng.choice(["bf16", "fp32"]), residual=rng.random() < 0.5, bias=rng.random() < 0.6, train=rng.random() < 0.7)
    if kind in ("scan", "step"):
        step = rng.choice([64, 8, 1])
        channels = max(step, _log_int(rng, 8, MAX_CHANNELS) // step * step)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        if kind == "step":
            return dict(kind=kind, sequences=_log_int(rng, 1, MAX_SEQUENCES), channels=channels, dtype=dtype)
        tokens = _log_int(rng, 1, MAX_LENGTH)
        sequences = min(tokens, _log_int(rng, 1, 64))
        packed = rng.random() < 0.5
        return dict(kind=kind, sequences=sequences, tokens=tokens if packed else tokens // sequences * sequences, packed=packed, channels=channels,
                    dtype=dtype, joint=rng.random() < 0.4, state=rng.random() < 0.5, train=rng.random() < 0.7)
    experts = rng.choice([8, 16, 60, 64, 128, 160, 256, MAX_EXPERTS])
    step = rng.choice([64, 8])
    ranks = rng.choice([r for r in (1, 2, 4, 8) if experts % r == 0])
    return dict(kind=kind, tokens=_log_int(rng, 1, 32768), hidden=max(step, _log_int(rng, 64, 7168) // step * step), experts=experts,
                top_k=rng.randint(1, MAX_TOPK if experts > 8 else 6), ranks=ranks, renormalize=rng.random() < 0.7,
                masked=rng.choice([0.0, 0.0, 0.3]), train=rng.random() < 0.7)


def draw(rng):
    """One more case of the same ranges, never more work than the largest listed one of its kind."""
    limit = {}
    for c in listed():
        w = work(c)
        have = limit.get(c["kind"], (0, 0))
        limit[c["kind"]] = (max(have[0], w["bytes"]), max(have[1], w["flops"]))
    limit["step"] = limit["scan"]
    while True:
        case = _draw_once(rng)
        w, (most_bytes, most_flops) = work(case), limit[case["kind"]]
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _normal(gen, *shape, std=1.0, mean=0.0):
    return torch.empty(*shape, device="cuda").normal_(mean, std, generator=gen)


def _uniform(gen, *shape, lo=0.0, hi=1.0):
    return torch.empty(*shape, device="cuda").uniform_(lo, hi, generator=gen)


def _prepare_norm(c, gen):
    R, H, t = c["rows"], c["hidden"], _type(c["dtype"])
    # activations: channels of very different sizes, some of them far from zero
    size, middle = _normal(gen, H).exp_(), _normal(gen, H, std=0.5)
    rows = lambda: (_normal(gen, R, H) * size + middle).to(t)
    s = {"case": dict(c), "x": rows(), "weight": _normal(gen, H, mean=1.0, std=0.2).to(_type(c["weights"]))}
    if c["bias"]:
        s["bias"] = _normal(gen, H, std=0.2).to(_type(c["weights"]))
    if c["residual"]:
        s["residual"] = rows()
    if c["train"]:
        for name in ("x", "weight", "bias", "residual"):
            if name in s:
                s[name].requires_grad_(True)
        s["dy"] = _normal(gen, R, H).to(t)
        if c["residual"]:
            s["dsum"] = _normal(gen, R, H).to(t)
    return s


def _lengths(c):
    """The sequences' lengths: all alike, or those of packed documents (they add up to ``tokens`` at most, empty ones and single
    tokens among them)."""
    S = c["sequences"]
    if not c["packed"]:
        return [c["tokens"] // S] * S
    rng = random.Random("%d %d" % (S, c["tokens"]))
    share = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(S)]
    lengths = [int(c["tokens"] * s / sum(share)) for s in share]
    if S > 3:
        small = rng.sample(range(S), 3)
        for i, n in zip(small, (0, 1, 0)):
            lengths[i] = min(lengths[i], n)
    return lengths


def _offsets(c):
    at = [0]
    for n in _lengths(c):
        at.append(at[-1] + n)
    return at


def _rows(c):
    # (packed batches are padded to a multiple of 64 rows, behind the last sequence)
    return (c["tokens"] + 63) // 64 * 64 if c["packed"] else c["tokens"]


def _prepare_scan(c, gen):
    D, t = c["channels"], _type(c["dtype"])
    S = c["sequences"]
    N = S if c["kind"] == "step" else _rows(c)
    # channels that forget at once beside channels that remember for thousands of tokens
    centre = _uniform(gen, D, lo=-1.0, hi=8.0)
    s = {"case": dict(c)}
    if c.get("joint"):
        both = torch.cat([_normal(gen, N, D), _normal(gen, N, D) + centre], dim=1).to(t)
        s["x"], s["gate"] = both[:, :D], both[:, D:]
    else:
        s["x"], s["gate"] = _normal(gen, N, D).to(t), (_normal(gen, N, D) + centre).to(t)
    if c["kind"] == "step":
        s["state"] = _normal(gen, S, D, std=0.5)
        return s
    shape = (N, D) if c["packed"] else (S, N // S, D)
    for name in ("x", "gate"):
        s[name] = s[name].view(shape)
    if c["packed"]:
        s["offsets"] = torch.tensor(_offsets(c), dtype=torch.int32, device="cuda")
    if c["state"]:
        s["initial"] = _normal(gen, S, D, std=0.5)
    if c["train"]:
        for name in ("x", "gate", "initial"):
            if name in s:
                s[name].requires_grad_(True)
        s["dh"] = _normal(gen, *shape).to(t)
        if c["state"]:
            s["dfinal"] = _normal(gen, S, D)
    return s


def _prepare_route(c, gen):
    T, H, E, K = c["tokens"], c["hidden"], c["experts"], c["top_k"]
    s = {"case": dict(c)}
    s["w_gate"] = _normal(gen, E, H, std=1.5 / math.sqrt(H)).to(torch.bfloat16)
    # a common direction makes some experts popular
    common = _normal(gen, H, std=0.5)
    x = (_normal(gen, T + T // 4 + 64, H) + common).to(torch.bfloat16)
    top = (x.float() @ s["w_gate"].float().t()).sort(dim=1, descending=True).values[:, :K + 1]
    close = (top[:, :-1] - top[:, 1:]).amin(dim=1) < GAP if top.shape[1] > 1 else torch.zeros(len(x), dtype=torch.bool, device="cuda")
    s["x"] = x[close.int().sort(stable=True).indices[:T]].contiguous()
    if c["masked"] > 0:
        s["mask"] = _uniform(gen, T) >= c["masked"]
    if c["train"]:
        s["x"].requires_grad_(True)
        s["w_gate"].requires_grad_(True)
        s["dweights"] = _normal(gen, T, K, std=1.0 / T)
        s["dbalance"], s["dz"] = torch.full((), 0.01, device="cuda"), torch.full((), 0.001, device="cuda")
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"norm": _prepare_norm, "scan": _prepare_scan, "step": _prepare_scan, "route": _prepare_route}[case["kind"]](case, gen)


# ---------------------------------------------------------------------------------------------------------------------
# one pass, in its plain form
# ---------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    total = s["x"].float() + s["residual"].float() if c["residual"] else s["x"].float()
    centred = total - total.mean(dim=1, keepdim=True)
    rstd = (centred.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    unit = centred * rstd
    weight = s["weight"].float()
    y = unit * weight
    if c["bias"]:
        y = y + s["bias"].float()
    got = {"y": y.to(t)}
    if c["residual"]:
        got["sum"] = total.to(t)
    if not c["train"]:
        return got
    dy = s["dy"].float()
    d = dy * weight
    dx = rstd * (d - d.mean(dim=1, keepdim=True) - unit * (d * unit).mean(dim=1, keepdim=True))
    if c["residual"]:
        dx = dx + s["dsum"].float()
    got["dx"] = dx.to(t)
    got["dweight"] = (dy * unit).sum(dim=0).to(s["weight"].dtype)
    if c["bias"]:
        got["dbias"] = dy.sum(dim=0).to(s["bias"].dtype)
    if c["residual"]:
        got["dresidual"] = got["dx"]
    return got


def _doubled(a, b):
    """``y_t = a_t y_{t-1} + b_t`` along the first dimension from zero, in a logarithm of passes: after each, ``(a, b)`` of a row stand
    for twice as many rows up to it."""
    step = 1
    while step < len(a):
        b = torch.cat([b[:step], a[step:] * b[:-step] + b[step:]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _firsts(c, offsets):
    """First and last rows of the sequences that have any, and which these are."""
    live = [i for i, n in enumerate(_lengths(c)) if n > 0]
    return [offsets[i] for i in live], [offsets[i + 1] - 1 for i in live], live


@torch.no_grad()
def _plain_scan(s):
    c, t = s["case"], s["x"].dtype
    D, S, offsets = c["channels"], c["sequences"], _offsets(c)
    total = offsets[-1]
    x, gate = (s[n].reshape(-1, D)[:total].float() for n in ("x", "gate"))
    first, last, live = _firsts(c, offsets)
    keep = 1.0 / (1.0 + (-gate).exp())
    take = 1.0 / (1.0 + gate.exp())
    initial = s["initial"].float() if c["state"] else torch.zeros(S, D, device="cuda")
    a, b = keep.clone(), take * x
    b[first] += a[first] * initial[live]
    a[first] = 0.0
    h = _doubled(a, b) if total else b
    final = initial.clone()
    final[live] = h[last]

    def rows(v, kind=t):
        whole = torch.zeros(_rows(c), D, dtype=kind, device="cuda")
        whole[:total] = v
        return whole.view(s["x"].shape)

    got = {"h": rows(h)}
    if c["state"]:
        got["final"] = final
    if not c["train"]:
        return got
    # the gradient of h_t: its own, and what flows back through h_{t+1}
    dh = s["dh"].reshape(-1, D)[:total].float()
    dfinal = s["dfinal"].float() if c["state"] else torch.zeros(S, D, device="cuda")
    back = torch.cat([keep[1:], torch.zeros_like(keep[:1])]) if total else keep
    g = dh.clone()
    back[last] = 0.0
    g[last] += dfinal[live]
    if total:
        g = _doubled(back.flip(0), g.flip(0)).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]]) if total else h
    before[first] = initial[live]
    got["dx"] = rows(take * g)
    got["dgate"] = rows(g * keep * take * (before - x))
    if c["state"]:
        got["dinitial"] = dfinal.clone()
        got["dinitial"][live] = keep[first] * g[first]
    return got


@torch.no_grad()
def _plain_step(s):
    x, gate = s["x"].float(), s["gate"].float()
    s["state"].copy_(s["state"] / (1.0 + (-gate).exp()) + x / (1.0 + gate.exp()))
    return s["state"].to(s["x"].dtype), s["state"]


@torch.no_grad()
def _plain_route(s):
    c = s["case"]
    T, E, K = c["tokens"], c["experts"], c["top_k"]
    x, w_gate = s["x"].float(), s["w_gate"].float()
    logits = x @ w_gate.t()
    shifted = logits - logits.max(dim=1, keepdim=True).values
    total = shifted.exp().sum(dim=1, keepdim=True)
    probs = shifted.exp() / total
    lse = (logits.max(dim=1, keepdim=True).values + total.log()).squeeze(1)
    idx = probs.sort(dim=1, descending=True, stable=True).indices[:, :K]
    chosen = probs.gather(1, idx)
    weights = chosen / chosen.sum(dim=1, keepdim=True) if c["renormalize"] else chosen
    expert = torch.arange(E, device="cuda")
    per_rank = E // c["ranks"]
    in_rank = (idx.unsqueeze(2) // per_rank == torch.arange(c["ranks"], device="cuda")).any(dim=1)
    live = s["mask"].float() if "mask" in s else torch.ones(T, device="cuda")
    n = live.sum()
    share = torch.where(n > 0, 1.0 / n, 0.0)
    hits = torch.zeros(T, E, device="cuda").scatter_(1, idx, 1.0) * live.unsqueeze(1)
    counts = hits.sum(dim=0, dtype=torch.float64)
    load = (counts * (E / K)).float() * share
    balance = (load * ((probs * live.unsqueeze(1)).sum(dim=0) * share)).sum()
    z_loss = (lse.square() * live).sum() * share
    got = {"idx": idx, "weights": weights, "in_rank": in_rank, "balance": balance, "z": z_loss, "counts": counts.long()}
    if not c["train"]:
        return got
    up = s["dweights"]
    if c["renormalize"]:
        at_chosen = weights * (up - (up * weights).sum(dim=1, keepdim=True))
        dlogits = torch.zeros_like(probs).scatter_(1, idx, at_chosen)
    else:
        dp = torch.zeros_like(probs).scatter_(1, idx, up)
        dlogits = probs * (dp - (dp * probs).sum(dim=1, keepdim=True))
    spread = probs * (load - (probs * load).sum(dim=1, keepdim=True))
    dlogits = dlogits + (s["dbalance"] * share) * live.unsqueeze(1) * spread
    dlogits = dlogits + (2.0 * s["dz"] * share) * (live * lse).unsqueeze(1) * probs
    got["dx"] = (dlogits @ w_gate).to(torch.bfloat16)
    got["dw_gate"] = (dlogits.t() @ x).to(torch.bfloat16)
    return got


# ---------------------------------------------------------------------------------------------------------------------
# one pass, through the framework
# ---------------------------------------------------------------------------------------------------------------------
def _own_norm(s):
    from streamep_b200.ops import layer_norm
    c = s["case"]
    names = [n for n in ("x", "weight", "bias", "residual") if n in s]
    with torch.set_grad_enabled(c["train"]):
        out = layer_norm(s["x"], s["weight"], s.get("bias"), eps=EPS, residual=s.get("residual"))
    y, total = out if c["residual"] else (out, None)
    got = {"y": y.detach()}
    if c["residual"]:
        got["sum"] = total.detach()
    if c["train"]:
        outs, ups = ((y, total), (s["dy"], s["dsum"])) if c["residual"] else ((y,), (s["dy"],))
        for n, g in zip(names, torch.autograd.grad(outs, [s[n] for n in names], ups)):
            got["d" + n] = g
    return got


def _own_scan(s):
    from streamep_b200.ops import gated_scan
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        out = gated_scan(s["x"], s["gate"], initial_state=s.get("initial"), offsets=s.get("offsets"), return_state=c["state"])
    h, final = out if c["state"] else (out, None)
    got = {"h": h.detach()}
    if c["state"]:
        got["final"] = final.detach()
    if c["train"]:
        names = ["x", "gate"] + (["initial"] if c["state"] else [])
        outs, ups = ((h, final), (s["dh"], s["dfinal"])) if c["state"] else ((h,), (s["dh"],))
        for n, g in zip(names, torch.autograd.grad(outs, [s[n] for n in names], ups)):
            got["d" + n] = g
    return got


def _own_step(s):
    from streamep_b200.ops import gated_scan_step_
    return gated_scan_step_(s["state"], s["x"], s["gate"]), s["state"]


def _own_route(s):
    from streamep_b200.ops import balanced_router
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        r = balanced_router(s["x"], s["w_gate"], c["top_k"], num_ranks=c["ranks"], renormalize=c["renormalize"], mask=s.get("mask"))
    got = {"idx": r.topk_idx, "weights": r.topk_weights.detach(), "in_rank": r.is_token_in_rank, "balance": r.balance_loss.detach(),
           "z": r.z_loss.detach(), "counts": r.expert_counts}
    if c["train"]:
        got["dx"], got["dw_gate"] = torch.autograd.grad((r.topk_weights, r.balance_loss, r.z_loss), (s["x"], s["w_gate"]),
                                                        (s["dweights"], s["dbalance"], s["dz"]))
    return got


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"norm": _own_norm, "scan": _own_scan, "step": _own_step, "route": _own_route}[kind](s)
    return {"norm": _plain_norm, "scan": _plain_scan, "step": _plain_step, "route": _plain_route}[kind](s)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _exact_norm(c, s):
    leaf = {n: s[n].detach().double().requires_grad_(True) for n in ("x", "weight", "bias", "residual") if n in s}
    total = leaf["x"] + leaf["residual"] if c["residual"] else leaf["x"]
    var, mean = torch.var_mean(total, dim=-1, correction=0, keepdim=True)
    y = torch.addcmul(leaf["bias"] if c["bias"] else torch.zeros((), dtype=torch.float64, device="cuda"),
                      (total - mean) / torch.sqrt(var + EPS), leaf["weight"])
    got = {"y": y.detach()}
    if c["residual"]:
        got["sum"] = total.detach()
    if c["train"]:
        value = (y * s["dy"].double()).sum()
        if c["residual"]:
            value = value + (total * s["dsum"].double()).sum()
        grads = dict(zip(leaf, torch.autograd.grad(value, list(leaf.values()))))
        for n in ("x", "weight", "bias", "residual"):
            if n in grads:
                got["d" + n] = grads[n]
    return got


def _blocks(a, b, start):
    """``y_t = a_t y_{t-1} + b_t`` from ``start`` (all rows of one sequence): the rows of equally long blocks one after another, all
    blocks at once, first from zero, then from what the block before ends with."""
    n, D = a.shape
    length = max(1, math.isqrt(n))
    count = -(-n // length)
    pad = count * length - n
    if pad:
        a = torch.cat([a, a.new_ones(pad, D)])
        b = torch.cat([b, b.new_zeros(pad, D)])
    a, b = a.view(count, length, D), b.view(count, length, D)
    end, factor = torch.zeros_like(b[:, 0]), torch.ones_like(a[:, 0])
    for i in range(length):
        end, factor = a[:, i] * end + b[:, i], factor * a[:, i]
    carry = torch.empty_like(end)
    now = start
    for k in range(count):
        carry[k] = now
        now = factor[k] * now + end[k]
    y = torch.empty_like(b)
    for i in range(length):
        carry = a[:, i] * carry + b[:, i]
        y[:, i] = carry
    return y.view(-1, D)[:n]


@torch.no_grad()
def _exact_scan(c, s):
    D, S, offsets = c["channels"], c["sequences"], _offsets(c)
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")
    x, gate = s["x"].reshape(-1, D).double(), s["gate"].reshape(-1, D).double()
    initial = s["initial"].double() if c["state"] else zeros(S, D)
    h, final = zeros(_rows(c), D), initial.clone()
    if c["train"]:
        dh = s["dh"].reshape(-1, D).double()
        dfinal = s["dfinal"].double() if c["state"] else zeros(S, D)
        dx, dgate, dinitial = zeros(_rows(c), D), zeros(_rows(c), D), dfinal.clone()
    for i in range(S):
        p, q = offsets[i], offsets[i + 1]
        if p == q:
            continue
        keep, take = torch.sigmoid(gate[p:q]), torch.sigmoid(-gate[p:q])
        h[p:q] = _blocks(keep, take * x[p:q], initial[i])
        final[i] = h[q - 1]
        if not c["train"]:
            continue
        # what flows back into row t is keep_{t+1} times the whole gradient of row t + 1
        own_part = dh[p:q].flip(0).clone()
        own_part[0] += dfinal[i]
        through = torch.cat([zeros(1, D), keep.flip(0)[:-1]])
        g = _blocks(through, own_part, zeros(D)).flip(0)
        previous = torch.cat([initial[i][None], h[p:q - 1]])
        dx[p:q] = g * take
        dgate[p:q] = g * (previous - x[p:q]) * keep * take
        dinitial[i] = g[0] * keep[0]
    shape = s["x"].shape
    got = {"h": h.view(shape)}
    if c["state"]:
        got["final"] = final
    if c["train"]:
        got["dx"], got["dgate"] = dx.view(shape), dgate.view(shape)
        if c["state"]:
            got["dinitial"] = dinitial
    return got


@torch.no_grad()
def _exact_step(c, s):
    keep = torch.sigmoid(s["gate"].double())
    h = torch.lerp(s["x"].double(), s["state"].double(), keep)
    return h, h


def _exact_route(c, s):
    T, E, K = c["tokens"], c["experts"], c["top_k"]
    x, w_gate = (s[n].detach().double().requires_grad_(True) for n in ("x", "w_gate"))
    logits = torch.einsum("th,eh->te", x, w_gate)
    probs = torch.softmax(logits, dim=1)
    idx = torch.argsort(logits.detach(), dim=1, descending=True, stable=True)[:, :K]
    weights = torch.softmax(logits.gather(1, idx), dim=1) if c["renormalize"] else probs.gather(1, idx)
    counted = s["mask"] if "mask" in s else torch.ones(T, dtype=torch.bool, device="cuda")
    counts = torch.bincount(idx[counted].reshape(-1), minlength=E)
    n = max(1, int(counted.sum()))
    balance = E * torch.dot(counts.double() / (K * n), probs[counted].sum(dim=0) / n)
    z = torch.logsumexp(logits[counted], dim=1).square().sum() / n
    in_rank = torch.zeros(T, c["ranks"], dtype=torch.bool, device="cuda")
    in_rank[torch.arange(T, device="cuda")[:, None], idx // (E // c["ranks"])] = True
    got = {"idx": idx, "weights": weights.detach(), "in_rank": in_rank, "balance": balance.detach(), "z": z.detach(), "counts": counts}
    if c["train"]:
        value = (weights * s["dweights"].double()).sum() + balance * s["dbalance"].double() + z * s["dz"].double()
        got["dx"], got["dw_gate"] = torch.autograd.grad(value, (x, w_gate))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "scan": _exact_scan, "step": _exact_step, "route": _exact_route}[case["kind"]](case, s)


def work(case):
    c = case
    if c["kind"] == "route":
        T, H, E, K = c["tokens"], c["hidden"], c["experts"], c["top_k"]
        values = 2.0 * (T + E) * H
        outs = T * (12.0 * K + c["ranks"]) + 8.0 * E + (T if c["masked"] > 0 else 0.0)
        if not c["train"]:
            return {"bytes": values + outs, "flops": 2.0 * T * H * E}
        return {"bytes": 2.0 * values + outs + 4.0 * T * K, "flops": 6.0 * T * H * E}
    width = 2.0 if c["dtype"] == "bf16" else 4.0
    if c["kind"] == "norm":
        array, vector = width * c["rows"] * c["hidden"], (2.0 if c["weights"] == "bf16" else 4.0) * c["hidden"] * (2 if c["bias"] else 1)
        arrays = 4 if c["residual"] else 2                 # x, residual; y, sum
        if c["train"]:
            arrays += 3 if c["residual"] else 2            # the gradients of y and sum; of x (the residual's is the same)
        return {"bytes": arrays * array + vector * (2 if c["train"] else 1), "flops": (20.0 if c["train"] else 8.0) * c["rows"] * c["hidden"]}
    if c["kind"] == "step":
        count = float(c["sequences"] * c["channels"])
        return {"bytes": count * (3.0 * width + 8.0), "flops": 6.0 * count}
    count = float(_rows(c) * c["channels"])
    states = 4.0 * c["sequences"] * c["channels"] * ((4 if c["train"] else 2) if c["state"] else 0)
    return {"bytes": width * count * (6 if c["train"] else 3) + states, "flops": (18.0 if c["train"] else 6.0) * count}
