"""Gradients of the normalisation and of trained routing against differences of their formulas in 64 bits, along the direction in which the slope is largest:
the signs of the gradient, so that the slope is the sum of its magnitudes.  The differences' own error is of second order: from twice the
step it is a third of the change.  The gradient's is the element-wise bound of the operators' tests, summed; each test says how small a part of the slope
both are, so that a gradient that is missing a term, or has a wrong sign, cannot pass."""
import pytest
import torch

from streamep_b200.ops import balanced_router, layer_norm, rms_norm

gpu = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
ULP = 2.0 ** -24


def against_differences(value, at, grad, slack, step, most):
    """`value` of tensors `at` (64 bits), its gradient with respect to the one that `at` yields for a shift; `most`: what the errors may be of the slope."""
    v = torch.sign(grad.double())
    slope = float((grad.double() * v).sum())
    exact, twice = ((value(at(k * step * v)) - value(at(-k * step * v))) / (2 * k * step) for k in (1, 2))
    bound = float(slack.sum()) + abs(twice - exact)
    assert bound <= most * slope, (bound, slope)
    assert abs(slope - exact) <= bound, (slope, exact, bound)


def norm_value(center):
    def value(p):
        s = p["x"] + p["residual"]
        c = s - s.mean(-1, keepdim=True) if center else s
        u = c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        y = u * p["weight"] + p.get("bias", 0.0)
        return float((y * p["dy"]).sum() + (s * p["dsum"]).sum())
    return value


@gpu
@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("H", [64, 1001, 2048, 9000])
def test_normalisation(native, H, center):
    g = torch.Generator(device=DEV).manual_seed(H)
    rows = 3
    matrix = lambda: torch.randn(rows, H, generator=g, device=DEV)
    t = {"x": matrix() * 1.5 + 0.7, "residual": matrix(), "weight": 1 + 0.3 * torch.randn(H, generator=g, device=DEV)}
    if center:
        t["bias"] = 0.3 * torch.randn(H, generator=g, device=DEV)
    dy, dsum = matrix(), matrix()
    leaves = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    f = (lambda x, w, **kw: layer_norm(x, w, leaves["bias"], **kw)) if center else rms_norm
    out = f(leaves["x"], leaves["weight"], eps=1e-5, residual=leaves["residual"])
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), [dy, dsum])))
    d64 = {n: v.double() for n, v in {**t, "dy": dy, "dsum": dsum}.items()}
    # the bounds of tests/test_layer_norm.py
    K = 48 + H / 32
    s = d64["x"] + d64["residual"]
    mean = s.mean(-1, keepdim=True) if center else 0.0 * s[:, :1]
    rstd = ((s - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    U = 1 + (s.abs() + s.abs().mean(-1, keepdim=True)) * rstd
    d = (d64["dy"] * d64["weight"]).abs()
    slack_x = K * ULP * rstd * (d + d.mean(-1, keepdim=True) + U * (d * U).mean(-1, keepdim=True)) + ULP * d64["dsum"].abs()
    more = (K + 160 + rows / 8) * ULP
    slack = {"x": slack_x, "residual": slack_x, "weight": more * (d64["dy"].abs() * U).sum(0), "bias": more * d64["dy"].abs().sum(0)}
    for n in t:
        at = lambda shift: {**d64, n: d64[n] + shift}
        against_differences(norm_value(center), at, grads[n], slack[n] + ULP * grads[n].double().abs(), 2.0 ** -12, 0.01)


@gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,K", [(16, 3), (160, 6)])
def test_routing(native, E, K, renormalize):
    T, H = 40, 64
    g = torch.Generator(device=DEV).manual_seed(E)
    x = (torch.randint(-16, 17, (T, H), generator=g, device=DEV) / 16.0).to(torch.bfloat16)
    w = (torch.randint(-16, 17, (E, H), generator=g, device=DEV) / 32.0).to(torch.bfloat16)
    up, db, dzl = torch.randn(T, K, generator=g, device=DEV), 20.0, 5.0
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = balanced_router(xl, wl, K, renormalize=renormalize)
    grads = torch.autograd.grad([r.topk_weights, r.balance_loss, r.z_loss], [xl, wl], [up, torch.tensor(db, device=DEV), torch.tensor(dzl, device=DEV)])
    idx, load = r.topk_idx, r.expert_counts.double() * E / (K * T)

    def value(p):                                        # with the choice held, as the gradient has it
        z = p[0] @ p[1].t()
        prob = torch.softmax(z, 1)
        c = prob.gather(1, idx)
        c = c / c.sum(1, keepdim=True) if renormalize else c
        return float((c * up.double()).sum() + db * (load * prob.mean(0)).sum() + dzl * torch.logsumexp(z, 1).square().mean())
    a, b = x.double(), w.double()
    z = a @ b.t()
    prob, lse = torch.softmax(z, 1), torch.logsumexp(z, 1)
    c = prob.gather(1, idx)
    c = c / c.sum(1, keepdim=True) if renormalize else c
    size = (c * up.double().abs()).sum(1, keepdim=True)
    D = torch.zeros_like(prob).scatter_add_(1, idx, c * up.double().abs()) + (prob if not renormalize else torch.zeros_like(prob).scatter_(1, idx, c)) * size
    D = D + abs(db) / T * prob * (load + (prob * load).sum(1, keepdim=True)) + 2 * abs(dzl) / T * lse.abs()[:, None] * prob
    # dz: two bf16 numbers, or one; what it is made of (tests/test_balanced_router.py); 17 2^-23 for each step of 16 that an accumulator takes, for each of the two
    P = (E / 32 + 14 + 2 * float(z.abs().max())) * ULP
    dz, layers = (2.0 ** -16, 2) if E <= 128 else (2.0 ** -8, 1)
    rel = lambda n: dz + 4 * P + (T / 16 + 160) * ULP + layers * -(-n // 16) * 17 * 2.0 ** -23
    for i, (grad, size, n) in enumerate(((grads[0], D @ b.abs(), E), (grads[1], D.t() @ a.abs(), T))):
        at = lambda shift: (a + shift, b) if i == 0 else (a, b + shift)
        against_differences(value, at, grad, rel(n) * size + 2.0 ** -8 * grad.double().abs(), 2.0 ** -12, 0.02 if E <= 128 else 0.05)
