"""layer_norm and rms_norm against 64-bit arithmetic: types, row lengths around vectors and blocks, strides and places off every
boundary, few and many rows, the residual stream, each subset of gradients, non-finite rows, streams, captured graphs, refusals.

Tolerances.  With n additions in a row (a thread's H / 32 at most, its warp's and its block's) a mean is off by (n + 2) 2^-24 of the
mean magnitude, a centred value u / rstd by that and its own rounding, the deviation by (n + 8) / 2 2^-24 of itself: K 2^-24 of
U = 1 + (|s| + mean |s|) rstd bounds u's error with K = 48 + H / 32.  y multiplies and adds (two more roundings, within K), dx is formed of d, mean d
and u mean(d u), each with those errors.  A sum over rows adds its own additions, at most rows / 8 + 160.  What is returned in
fewer bits is rounded once: eps / 2 of the value."""
import pytest
import torch

from streamep_b200.ops import layer_norm, rms_norm

gpu = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
ULP = 2.0 ** -24


def make(rows, H, dtype, wdtype, seed=0, bias=True, residual=True, grad=True, pad=0, off=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def matrix():
        flat = torch.randn(off + max(rows, 1) * (H + pad), generator=g, device=DEV) * 1.5 + 0.7
        return flat.to(dtype)[off:off + rows * (H + pad)].view(rows, H + pad)[:, :H]
    t = {"x": matrix(), "weight": (1.0 + 0.3 * torch.randn(H, generator=g, device=DEV)).to(wdtype)}
    if bias:
        t["bias"] = (0.3 * torch.randn(H, generator=g, device=DEV)).to(wdtype)
    if residual:
        t["residual"] = matrix()
    if grad:
        for v in t.values():
            v.requires_grad_(True)
    return t, torch.randn(rows, H, generator=g, device=DEV).to(dtype), torch.randn(rows, H, generator=g, device=DEV).to(dtype)


def call(t, center, eps=1e-5):
    f = (lambda x, w, **kw: layer_norm(x, w, t.get("bias"), **kw)) if center else rms_norm
    out = f(t["x"], t.get("weight"), eps=eps, residual=t.get("residual"))
    return out if t.get("residual") is not None else (out, None)


def half_step(want, dtype):
    return want.abs() * (torch.finfo(dtype).eps / 2) if dtype != F32 else want.abs() * 2.0 ** -24


def near(got, want, slack, what):
    over = (got.double() - want).abs() - (slack + half_step(want, got.dtype))
    assert got.shape == want.shape and bool((over <= 0).all()), f"{what}: {float(over.max()):.3e} above the bound"


def check(t, center, dy=None, dsum=None, eps=1e-5, grads=True):
    y, total = call(t, center, eps)
    H = y.shape[-1]
    K = 48 + H / 32
    d64 = {n: v.detach().double() for n, v in t.items()}
    s = d64["x"] + d64["residual"] if "residual" in t else d64["x"]
    mean = s.mean(-1, keepdim=True) if center else torch.zeros_like(s[..., :1])
    rstd = ((s - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    w = d64.get("weight", torch.ones(H, dtype=torch.float64, device=DEV))
    b = d64.get("bias", torch.zeros(H, dtype=torch.float64, device=DEV))
    u = (s - mean) * rstd
    U = 1 + (s.abs() + s.abs().mean(-1, keepdim=True)) * rstd
    near(y, u * w + b, K * ULP * (U * w.abs() + b.abs()), "y")
    assert y.dtype == t["x"].dtype
    if total is not None:
        near(total, s, 0.0 * s, "sum")
    if not grads:
        return y, total
    outs, ups = [y], [dy]
    if total is not None and dsum is not None:
        outs, ups = [y, total], [dy, dsum]
    got = dict(zip(t, torch.autograd.grad(outs, list(t.values()), ups)))
    d = dy.double() * w
    mean_d = d.mean(-1, keepdim=True) if center else 0.0
    dx = rstd * (d - mean_d - u * (d * u).mean(-1, keepdim=True))
    slack = K * ULP * rstd * (d.abs() + d.abs().mean(-1, keepdim=True) + U * (d.abs() * U).mean(-1, keepdim=True))
    if total is not None and dsum is not None:
        dx = dx + dsum.double()
        slack = slack + ULP * dsum.double().abs()
    near(got["x"], dx, slack, "dx")
    if "residual" in t:
        assert torch.equal(got["residual"], got["x"])
    flat = lambda v: v.reshape(-1, H)
    more = (K + 160 + flat(dy).shape[0] / 8) * ULP
    if "weight" in t:
        near(got["weight"], flat(dy.double() * u).sum(0), more * flat(dy.double().abs() * U).sum(0), "dweight")
        assert got["weight"].dtype == t["weight"].dtype
    if "bias" in t:
        near(got["bias"], flat(dy.double()).sum(0), more * flat(dy.double().abs()).sum(0), "dbias")
    return y, total


WIDTHS = [1, 2, 7, 8, 31, 33, 64, 100, 256, 264, 1000, 1001, 2048, 2056, 4096, 4097, 5120, 8192, 8193, 8200, 20000, 33000]


@gpu
@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("H", WIDTHS)
def test_widths(native, H, dtype, wdtype, center):
    for rows, residual in ((1, True), (5, False), (67, True)):
        t, dy, dsum = make(rows, H, dtype, wdtype, seed=H, residual=residual, bias=center)
        check(t, center, dy, dsum)


@gpu
@pytest.mark.parametrize("rows", [0, 1, 2, 147, 149, 1777, 5000])
@pytest.mark.parametrize("H,dtype", [(264, BF), (1001, F32), (96, F32), (2048, BF)])
def test_rows(native, rows, H, dtype):
    t, dy, dsum = make(rows, H, dtype, dtype, seed=rows)
    check(t, True, dy, dsum)


@gpu
@pytest.mark.parametrize("pad,off", [(8, 0), (3, 0), (0, 1), (1, 3), (16, 8)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_places(native, pad, off, dtype):
    t, dy, dsum = make(41, 512, dtype, dtype, seed=1, pad=pad, off=off, grad=False)
    t = {n: v.requires_grad_(True) for n, v in t.items()}
    check(t, True, dy, dsum)
    w = torch.randn(513, device=DEV).to(dtype)[1:].requires_grad_(True)       # a weight off every boundary
    check({**t, "weight": w}, True, dy, dsum)
    wide = torch.randn(41, 1024, device=DEV).to(dtype)
    check(t, True, wide[:, 1::2], wide[:, 512:])                            # upstream gradients with gaps
    column = torch.randn(512, 41, device=DEV).to(dtype).t().requires_grad_(True)
    check({**t, "x": column}, True, dy, dsum)


@gpu
def test_shapes(native):
    t, dy, dsum = make(24, 128, BF, BF, seed=3)
    flat = check(t, True, dy, dsum)
    for shape in ((2, 3, 4, 128), (24, 1, 128)):
        u = {n: (v.detach().view(shape) if v.dim() == 2 else v.detach()).requires_grad_(True) for n, v in t.items()}
        got = check(u, True, dy.view(shape), dsum.view(shape))
        assert torch.equal(got[0].view(24, 128), flat[0]) and torch.equal(got[1].view(24, 128), flat[1])
    one = check({"x": torch.randn(64, device=DEV, requires_grad=True)}, True, torch.randn(64, device=DEV))
    assert one[0].shape == (64,)
    # a row that is the same for all: the residual's gradient is summed over what it was repeated for
    base = torch.randn(1, 128, device=DEV).to(BF).requires_grad_(True)
    y, s = layer_norm(t["x"], t["weight"], residual=base.expand(24, 128))
    gx, gb = torch.autograd.grad([y, s], [t["x"], base], [dy, dsum])
    near(gb, gx.double().sum(0, keepdim=True), 24 * ULP * gx.double().abs().sum(0, keepdim=True) + 0.0, "broadcast residual")


@gpu
@pytest.mark.parametrize("H", [264, 1001, 8200])
def test_subsets_of_gradients(native, H):
    t, dy, dsum = make(33, H, BF, BF, seed=5, grad=False)
    names = list(t)
    full = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    y, s = call(full, True)
    want = dict(zip(names, torch.autograd.grad([y, s], list(full.values()), [dy, dsum])))
    for mask in range(1, 16):
        part = {n: v.clone().requires_grad_(bool(mask >> i & 1)) for i, (n, v) in enumerate(t.items())}
        y, s = call(part, True)
        chosen = [n for n in names if part[n].requires_grad]
        outs, ups = ([y, s], [dy, dsum]) if s.requires_grad else ([y], [dy])
        for n, g in zip(chosen, torch.autograd.grad(outs, [part[n] for n in chosen], ups)):
            assert torch.equal(g, want[n]), (mask, n)
    # one output alone
    y, s = call(full, True)
    gx, gr = torch.autograd.grad(s, [full["x"], full["residual"]], dsum)
    assert torch.equal(gx, dsum) and torch.equal(gr, dsum)
    y, s = call(full, True)
    alone = torch.autograd.grad(y, full["x"], dy)[0]
    assert alone.shape == dy.shape and not torch.equal(alone, want["x"])
    no_weight = {k: v for k, v in full.items() if k != "weight"}
    check(no_weight, True, dy, dsum)
    check({"x": full["x"]}, True, dy)
    check({"x": full["x"]}, False, dy)


@gpu
@pytest.mark.parametrize("H", [64, 1001, 2048, 9000])
def test_against_differences(native, H):
    t, dy, _ = make(6, H, F32, F32, seed=7, residual=False)
    g = torch.Generator(device=DEV).manual_seed(8)
    grads = dict(zip(t, torch.autograd.grad(call(t, True)[0], list(t.values()), dy)))
    for n in t:
        v = torch.randn(t[n].shape, generator=g, device=DEV)
        h = 2.0 ** -7

        def value(step, f64):
            p = {k: q.detach() + (step * v if k == n else 0.0) for k, q in t.items()}
            if f64:
                q = {k: a.double() for k, a in p.items()}
                c = q["x"] - q["x"].mean(-1, keepdim=True)
                out = c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * q["weight"] + q["bias"]
            else:
                out = call(p, True)[0].double()
            return float((out * dy.double()).sum())
        slope = float((grads[n].double() * v.double()).sum())
        mine, exact = ((value(h, f) - value(-h, f)) / (2 * h) for f in (False, True))
        # y is off by K 2^-24 (U |w| + |b|) <= K 2^-24 x 16 here, in either direction, over 2 h; the slope's own error is smaller
        bound = (48 + H / 32) * ULP * 16 * float(dy.abs().sum()) / h
        assert abs(mine - exact) <= bound
        assert abs(slope - exact) <= bound + 0.05 * h * float((dy.abs().sum(0) if v.dim() == 1 else dy.abs() * v.abs().pow(3)).sum())


@gpu
def test_constant_rows_and_eps(native):
    for dtype in (BF, F32):
        for H in (1, 64, 1001, 9000):
            x = torch.full((3, H), 2.5, device=DEV, dtype=dtype)          # variance 0
            b = torch.randn(H, device=DEV)
            assert torch.equal(layer_norm(x, None, b), b.expand(3, H).to(dtype))
            assert bool(layer_norm(x, eps=0.0).isnan().all())
            near(rms_norm(x), (x.double() / (x.double().square() + 1e-6).sqrt()), (48 + H / 32) * ULP * torch.ones(3, H, dtype=torch.float64, device=DEV), "rms")
    # rows far from zero: the variance is taken around the mean
    t = {"x": (torch.randn(5, 4096, device=DEV) * 0.01 + 1000.0).requires_grad_(True)}
    check(t, True, torch.randn(5, 4096, device=DEV))


@gpu
@pytest.mark.parametrize("H", [256, 1001, 9000])
def test_non_finite_rows_stay_alone(native, H):
    for bad in (float("inf"), float("-inf"), float("nan")):
        t, dy, dsum = make(9, H, F32, F32, seed=11, grad=False)
        y0, s0 = call(t, True)
        x = t["x"].clone()
        x[4, H // 2] = bad
        y, s = call({**t, "x": x}, True)
        keep = torch.arange(9, device=DEV) != 4
        assert torch.equal(y[keep], y0[keep]) and torch.equal(s[keep], s0[keep])
        assert bool(y[4].isnan().all())
        xl = x.clone().requires_grad_(True)
        gx, = torch.autograd.grad(call({**t, "x": xl}, True)[0], xl, dy)
        assert bool(gx[keep].isfinite().all()) and bool(gx[4].isnan().all())


@gpu
def test_repeats_streams_and_graphs(native):
    t, dy, dsum = make(777, 2048, BF, F32, seed=13)

    def run():
        y, s = call(t, True)
        return [y.detach(), s.detach()] + list(torch.autograd.grad([y, s], list(t.values()), [dy, dsum]))
    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.no_grad():
        t["x"].mul_(0.5)
    want = run()
    for v in held:
        v.fill_(float("nan"))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@gpu
def test_refusals(native):
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    for f in (lambda: layer_norm(x.half()), lambda: layer_norm(x, torch.ones(63, device=DEV)), lambda: layer_norm(x, w.half()),
              lambda: layer_norm(x, w, torch.ones(64, device=DEV).to(BF)), lambda: layer_norm(x, w.cpu()), lambda: layer_norm(x, residual=x.detach()[:2]),
              lambda: layer_norm(x, residual=x.detach().to(BF)), lambda: layer_norm(x, eps=-1.0), lambda: layer_norm(x[:, :0]),
              lambda: layer_norm(x, torch.ones(1, 64, device=DEV)), lambda: rms_norm(torch.zeros((), device=DEV))):
        with pytest.raises(ValueError):
            f()
    y = layer_norm(x, w)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            layer_norm(torch.autograd.forward_ad.make_dual(x, x))
    # what was saved must not have changed; the sum, which a program may go on in, was not
    r = x.detach().clone()
    y, s = layer_norm(x, w, residual=r)
    with torch.no_grad():
        s.add_(1.0)
    torch.autograd.grad(y.sum(), x)
    y, s = layer_norm(x, w, residual=r)
    with torch.no_grad():
        r.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)


def test_refused_without_a_gpu():
    for f in (lambda: layer_norm(torch.ones(2, 8)), lambda: rms_norm(torch.ones(2, 8))):
        with pytest.raises(ValueError, match="CUDA"):
            f()
