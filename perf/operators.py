"""The end of a training step around the MoE layer, measured: the loss over the vocabulary, the norm of all gradients and
their clipping, and the optimizer's update.

Three kinds of call, each through the public entry points:

* ``loss``   ``linear_cross_entropy``: the output projection and the softmax cross entropy in one, without logits in
             memory; with ``train`` its gradients for the hidden states and for the projection
* ``clip``   ``clip_grad_norm_``: the global norm over a list of gradients, and their scaling where it is too large
* ``update`` ``grad_norm`` and ``adamw_step_``: the norm, and an AdamW update that applies the clipping on its way

Where ``own`` is false the same is computed in its plain form: 32-bit tensors, one elementary operation after another.
"""
import math
import random

import torch

own = False

#: Upper ends of the ranges that ``draw`` samples.
MAX_TOKENS, MAX_HIDDEN, MAX_VOCAB, MAX_TENSORS, MAX_ELEMENTS = 16384, 7168, 131072, 600, 400_000_000
IGNORED = -100
BETAS, EPS, DECAY, LEARNING_RATE = (0.9, 0.95), 1e-8, 0.1, 3e-4


def listed():
    return [
        # The benchmark's default layer below a vocabulary of ordinary size: a training step's loss and its gradients.
        dict(name="loss training", kind="loss", tokens=8192, hidden=2048, vocab=65536, train=True, reduction="mean",
             ignored=0.0, sharp=False),
        # The benchmark's wide layer below a large vocabulary: the largest call.
        dict(name="loss large vocabulary", kind="loss", tokens=8192, hidden=4096, vocab=128000, train=True,
             reduction="mean", ignored=0.0, sharp=True),
        # Ragged sizes, padded sequences (a quarter of the targets is ignored), a model that has learned something.
        dict(name="loss ragged", kind="loss", tokens=1777, hidden=1000, vocab=50257, train=True, reduction="mean",
             ignored=0.25, sharp=True),
        # Fine-tuning with a weight for each token (a policy gradient, distillation): the gradient of each token's loss.
        dict(name="loss per token", kind="loss", tokens=300, hidden=2048, vocab=100003, train=True, reduction="none",
             ignored=0.1, sharp=True),
        # The tiny layer of unit tests and debugging runs: launches and latency.
        dict(name="loss tiny", kind="loss", tokens=64, hidden=256, vocab=1000, train=True, reduction="mean",
             ignored=0.0, sharp=False),
        # Evaluation: the log-probability of every token of a held-out sequence, no gradient.
        dict(name="score sequence", kind="loss", tokens=4001, hidden=2048, vocab=100003, train=False, reduction="none",
             ignored=0.0, sharp=True),
        # The log-probability of one more token, as reranking asks for it: bound by reading the projection.
        dict(name="score one token", kind="loss", tokens=1, hidden=4096, vocab=128000, train=False, reduction="none",
             ignored=0.0, sharp=False),
        # Four of the default layers: few large gradients, a norm below the limit (the ordinary step of a stable run).
        dict(name="clip layers", kind="clip", layers=4, tensors=0, elements=0, layout="apart", dtype="bf16", over=False),
        # A long list of mixed gradients of every size, packed into flat buffers without alignment, above the limit.  The
        # backward pass that writes them is stood in for by one copy of each buffer.
        dict(name="clip packed list", kind="clip", layers=0, tensors=400, elements=30_000_001, layout="packed",
             dtype="mixed", over=True),
        # The list of a small model: launches and latency.
        dict(name="clip small list", kind="clip", layers=0, tensors=40, elements=200_003, layout="apart", dtype="fp32",
             over=False),
        # The default layers and their projection, bf16 weights with 32-bit master copies.
        dict(name="update layers", kind="update", layers=4, tensors=0, elements=0, layout="apart", dtype="bf16",
             master=True, step=100),
        # A list of odd sizes with 32-bit weights, the first step of a run.
        dict(name="update ragged list", kind="update", layers=0, tensors=250, elements=5_000_011, layout="packed",
             dtype="fp32", master=False, step=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(["loss", "clip", "update"], [6, 2, 2])[0]
    if kind == "loss":
        step = 64 if rng.random() < 0.6 else 8            # what the operator asks for: rows of whole 16-byte pieces
        hidden = max(step, _log_int(rng, 64, MAX_HIDDEN) // step * step)
        return dict(kind=kind, tokens=_log_int(rng, 1, MAX_TOKENS), hidden=hidden, vocab=_log_int(rng, 100, MAX_VOCAB),
                    train=rng.random() < 0.7, reduction=rng.choice(["mean", "mean", "sum", "none"]),
                    ignored=rng.choice([0.0, 0.0, 0.3]), sharp=rng.random() < 0.5)
    layers = rng.choice([0, 0, 0, 1, 2])
    case = dict(kind=kind, layers=layers, tensors=0 if layers else _log_int(rng, 1, MAX_TENSORS),
                elements=0 if layers else _log_int(rng, 1000, MAX_ELEMENTS), layout=rng.choice(["apart", "packed"]),
                dtype=rng.choice(["bf16", "fp32", "mixed"] if kind == "clip" else ["bf16", "fp32"]))
    if kind == "clip":
        case["over"] = rng.random() < 0.5
    else:
        case["master"] = case["dtype"] == "bf16" and rng.random() < 0.7
        case["step"] = rng.choice([1, 10, 1000])
    return case


def draw(rng):
    """One more case of the same ranges, never more work than the largest listed one of its kind."""
    limit = {}
    for c in listed():
        w = work(c)
        have = limit.get(c["kind"], (0, 0))
        limit[c["kind"]] = (max(have[0], w["bytes"]), max(have[1], w["flops"]))
    while True:
        case = _draw_once(rng)
        w, (most_bytes, most_flops) = work(case), limit[case["kind"]]
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """The lengths of a list of parameters: those of whole layers, or a ragged list (tiny and empty tensors among them)."""
    if case["layers"]:
        hidden, ffn, experts, vocab = 2048, 1408, 8, 65536
        layer = [experts * 2 * ffn * hidden, experts * hidden * ffn, experts * hidden, hidden]
        return layer * case["layers"] + ([vocab * hidden] if case["kind"] == "update" else [])
    rng = random.Random("%d %d" % (case["tensors"], case["elements"]))
    share = [math.exp(rng.gauss(0.0, 2.5)) for _ in range(case["tensors"])]
    sizes = [int(case["elements"] * s / sum(share)) for s in share]
    if len(sizes) > 3:
        sizes[rng.randrange(len(sizes))] = 0
        sizes[rng.randrange(len(sizes))] = 1
    return sizes


def _types(case, count):
    if case["dtype"] != "mixed":
        return [case["dtype"]] * count
    return ["fp32" if i % 4 == 3 else "bf16" for i in range(count)]


def _buffers(case, kinds, sizes):
    """One flat buffer for each type and the list's tensors in it: each from a place of its own, as an allocator gives
    it (the gaps hold zeros and stay so), or packed end to end."""
    whole, at, places = {}, {}, []
    for kind, n in zip(kinds, sizes):
        start = at.get(kind, 0)
        places.append(start)
        at[kind] = start + n if case["layout"] == "packed" else (start + n + 255) // 256 * 256
    for kind, n in at.items():
        whole[kind] = torch.zeros(n, dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
    return whole, [whole[k][p:p + n] for k, p, n in zip(kinds, places, sizes)]


def _lists(case, gen):
    sizes = _sizes(case)
    kinds = _types(case, len(sizes))
    grads, grad_list = _buffers(case, kinds, sizes)
    spread = random.Random(str(case["elements"]))
    for g in grad_list:
        g.normal_(0.0, 10.0 ** spread.uniform(-5.0, -2.5), generator=gen)
    s = {"case": dict(case), "grads": grads, "grad_list": grad_list}
    if case["kind"] == "clip":
        norm = math.sqrt(sum(float(g.float().square().sum()) for g in grads.values()))
        s["max_norm"] = norm * (0.3 if case["over"] else 3.0)
        if case["over"]:
            s["fresh"] = {k: g.clone() for k, g in grads.items()}
        return s
    s["step"], s["max_norm"] = case["step"], 0.5
    s["params"], s["param_list"] = _buffers(case, kinds, sizes)
    for kind in ["exp_avg", "exp_avg_sq"] + (["master"] if case["master"] else []):
        s[kind], s[kind + "_list"] = _buffers(case, ["fp32"] * len(sizes), sizes)
    for p in s["param_list"]:
        p.normal_(0.0, 0.02, generator=gen)
    if case["master"]:                                   # the weights are the master copies, rounded
        for m, p in zip(s["master_list"], s["param_list"]):
            m.copy_(p)
            m.add_(torch.empty_like(m).uniform_(-2e-5, 2e-5, generator=gen))
            p.copy_(m)
    if case["step"] > 1:
        for m, v, g in zip(s["exp_avg_list"], s["exp_avg_sq_list"], grad_list):
            m.copy_(g).mul_(0.3)
            v.copy_(g).square_().mul_(0.8)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] != "loss":
        return _lists(case, gen)
    T, H, V = case["tokens"], case["hidden"], case["vocab"]
    s = {"case": dict(case)}
    s["weight"] = torch.empty(V, H, dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.02, generator=gen)
    s["targets"] = torch.randint(0, V, (T,), generator=gen, device="cuda")
    x = torch.empty(T, H, device="cuda").normal_(0.0, 1.0, generator=gen)
    if case["sharp"]:                                    # the target's logit stands out by 0 to 12
        row = s["weight"][s["targets"]].float()
        x += row * (12.0 * torch.rand(T, 1, generator=gen, device="cuda") / row.square().sum(dim=1, keepdim=True))
    s["x"] = x.to(torch.bfloat16)
    if case["ignored"] > 0:
        s["targets"][torch.rand(T, generator=gen, device="cuda") < case["ignored"]] = IGNORED
        s["targets"][:1] = 0                             # one counts at least
    if case["train"]:
        s["upstream"] = (torch.randn(T, generator=gen, device="cuda") if case["reduction"] == "none"
                         else torch.ones((), device="cuda"))
        s["x"].requires_grad_(True)
        s["weight"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass, in its plain form
# ---------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def _plain_loss(s):
    c = s["case"]
    x, weight, targets = s["x"].float(), s["weight"].float(), s["targets"]
    counted = targets != IGNORED
    column = torch.where(counted, targets, 0).unsqueeze(1)
    logits = x @ weight.t()
    shifted = logits - logits.max(dim=1, keepdim=True).values
    log_prob = shifted - shifted.exp().sum(dim=1, keepdim=True).log()
    each = torch.where(counted, -log_prob.gather(1, column).squeeze(1), 0.0)
    share = 1.0 / counted.sum() if c["reduction"] == "mean" else torch.ones((), device=x.device)
    loss = each if c["reduction"] == "none" else each.sum() * share
    if not c["train"]:
        return loss
    scale = torch.where(counted, s["upstream"] * share, 0.0).unsqueeze(1)
    grad = log_prob.exp() * scale
    grad.scatter_add_(1, column, -scale)
    return loss, (grad @ weight).to(torch.bfloat16), (grad.t() @ x).to(torch.bfloat16)


def _plain_norm(grads):
    return torch.stack([g.float().square().sum() for g in grads.values()]).sum().sqrt()


@torch.no_grad()
def _plain_clip(s):
    norm = _plain_norm(s["grads"])
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g in s["grads"].values():
        g.copy_(g.float() * factor)
    return norm


@torch.no_grad()
def _plain_update(s):
    norm = _plain_norm(s["grads"])
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    (kind, params), = s["params"].items()
    g = s["grads"][kind].float() * factor
    m, v = s["exp_avg"]["fp32"], s["exp_avg_sq"]["fp32"]
    m.copy_(BETAS[0] * m + (1.0 - BETAS[0]) * g)
    v.copy_(BETAS[1] * v + (1.0 - BETAS[1]) * g * g)
    w = s["master"]["fp32"] if s["case"]["master"] else params.float()
    w = w * (1.0 - LEARNING_RATE * DECAY)
    w = w - LEARNING_RATE * (m / (1.0 - BETAS[0] ** s["step"])) / ((v / (1.0 - BETAS[1] ** s["step"])).sqrt() + EPS)
    if s["case"]["master"]:
        s["master"]["fp32"].copy_(w)
    params.copy_(w)
    return norm


# ---------------------------------------------------------------------------------------------------------------------
# one pass, through the framework
# ---------------------------------------------------------------------------------------------------------------------
def _own_loss(s):
    from streamep_b200.ops import linear_cross_entropy
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORED, reduction=c["reduction"])
    loss = linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORED, reduction=c["reduction"])
    return (loss.detach(),) + torch.autograd.grad(loss, (s["x"], s["weight"]), s["upstream"])


def _own_clip(s):
    from streamep_b200.ops import clip_grad_norm_
    return clip_grad_norm_(s["grad_list"], s["max_norm"])


def _own_update(s):
    from streamep_b200.ops import adamw_step_, grad_norm
    norm = grad_norm(s["grad_list"])
    adamw_step_(s["param_list"], s["grad_list"], s["exp_avg_list"], s["exp_avg_sq_list"],
                masters=s["master_list"] if s["case"]["master"] else None, step=s["step"], lr=LEARNING_RATE, betas=BETAS,
                eps=EPS, weight_decay=DECAY, norm=norm, max_norm=s["max_norm"])
    return norm


def run(s):
    c = s["case"]
    if c["kind"] == "loss":
        return _own_loss(s) if own else _plain_loss(s)
    if c["kind"] == "clip":
        if c["over"]:
            for kind, g in s["grads"].items():
                g.copy_(s["fresh"][kind])
        norm = _own_clip(s) if own else _plain_clip(s)
        return {"norm": norm, "grads": s["grads"]}
    norm = _own_update(s) if own else _plain_update(s)
    s["step"] += 1
    got = {"norm": norm, "params": s["params"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}
    if c["master"]:
        got["master"] = s["master"]
    return got


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def _exact_loss(case, s):
    T = case["tokens"]
    weight = s["weight"].double()
    live = s["targets"] != IGNORED
    weights = live.double()
    if case["reduction"] == "mean":
        weights /= weights.sum()
    if case["train"]:
        upstream = s["upstream"].double()
        dx = torch.zeros(T, case["hidden"], dtype=torch.float64, device="cuda")
        dweight = torch.zeros_like(weight)
    each = torch.zeros(T, dtype=torch.float64, device="cuda")
    rows = max(1, 200_000_000 // case["vocab"])
    for a in range(0, T, rows):
        b = min(T, a + rows)
        x = s["x"][a:b].double()
        z = torch.einsum("th,vh->tv", x, weight)
        lse = torch.logsumexp(z, dim=1)
        y = s["targets"][a:b].clamp(min=0)
        at = torch.arange(b - a, device="cuda")
        each[a:b] = (lse - z[at, y]) * weights[a:b]
        if case["train"]:
            p = torch.exp(z - lse[:, None])
            p[at, y] -= 1.0
            p *= (weights[a:b] * (upstream[a:b] if case["reduction"] == "none" else upstream))[:, None]
            dx[a:b] = torch.einsum("tv,vh->th", p, weight)
            dweight += torch.einsum("tv,th->vh", p, x)
    loss = each if case["reduction"] == "none" else each.sum()
    return (loss, dx, dweight) if case["train"] else loss


@torch.no_grad()
def _exact_lists(case, s):
    flat = {k: g.double() for k, g in s["grads"].items()}
    norm = math.sqrt(sum(float(torch.dot(g, g)) for g in flat.values()))
    scale = min(1.0, s["max_norm"] / (norm + 1e-6))
    value = torch.tensor(norm, dtype=torch.float64)
    if case["kind"] == "clip":
        return {"norm": value, "grads": {k: g * scale for k, g in flat.items()}}
    (kind, g), = flat.items()
    g = g * scale
    m = torch.lerp(g, s["exp_avg"]["fp32"].double(), BETAS[0])
    v = torch.lerp(g.square(), s["exp_avg_sq"]["fp32"].double(), BETAS[1])
    start = (s["master"]["fp32"] if case["master"] else s["params"][kind]).double()
    t = case["step"]
    denominator = v.sqrt() / math.sqrt(1.0 - BETAS[1] ** t) + EPS
    new = start - LEARNING_RATE * (DECAY * start + m / denominator / (1.0 - BETAS[0] ** t))
    got = {"norm": value, "params": {kind: new}, "exp_avg": {"fp32": m}, "exp_avg_sq": {"fp32": v}}
    if case["master"]:
        got["master"] = {"fp32": new}
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_loss(case, s) if case["kind"] == "loss" else _exact_lists(case, s)


def work(case):
    if case["kind"] == "loss":
        T, H, V = case["tokens"], case["hidden"], case["vocab"]
        values = 2.0 * T * H + 2.0 * V * H
        outs = 4.0 * (T if case["reduction"] == "none" else 1)
        if not case["train"]:
            return {"bytes": values + 8.0 * T + outs, "flops": 2.0 * T * H * V}
        return {"bytes": 2.0 * values + 8.0 * T + 2.0 * outs, "flops": 6.0 * T * H * V}
    sizes = _sizes(case)
    width = [2.0 if k == "bf16" else 4.0 for k in _types(case, len(sizes))]
    grads = sum(w * n for w, n in zip(width, sizes))
    count = float(sum(sizes))
    if case["kind"] == "clip":           # above the limit: the copy that stands in for the backward pass, and the scaling
        return {"bytes": grads * (4.0 if case["over"] else 1.0) + 4.0, "flops": 2.0 * count}
    held = 8.0 + (4.0 if case["master"] else 0.0)        # both moments, the master copy: read and written
    params = sum(w * n for w, n in zip(width, sizes))
    return {"bytes": grads + 2.0 * held * count + params * (1.0 if case["master"] else 2.0), "flops": 14.0 * count}
