"""linear_cross_entropy against the definition in 64 bits: sizes on both sides of every tile, ignored tokens, strides, refusals.

Tolerances.  Loss: a logit is an fp32 sum of H exact products (relative error of a few 2^-24 sqrt(H) of the sum of magnitudes, below 1e-6
of |x||w|), exponentials and logarithm add a few 2^-22: 2e-5 absolute on losses of order 1 to 20.  Gradients: dz is rounded to bf16
(2^-9 relative at most) and so is the result, independent errors: 2-norm within 2^-9 * sqrt(2) = 2.8e-3 of the result's, taken as 4e-3."""
import pytest
import torch

from streamep_b200 import StreamEPError
from streamep_b200.ops import linear_cross_entropy
from streamep_b200.ops import grouped_gemm as gg

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(T, H, V, seed=0, sharp=4.0, std=0.05):
    g = torch.Generator(device="cpu").manual_seed(seed)
    w = (torch.randn(V, H, generator=g) * std).to(torch.bfloat16)
    y = torch.randint(0, V, (T,), generator=g)
    x = torch.randn(T, H, generator=g)
    row = w[y].float()
    x = x + row * (sharp * torch.rand(T, 1, generator=g) / row.square().sum(1, keepdim=True))
    return x.to(torch.bfloat16).to(DEV), w.to(DEV), y.to(DEV)


def oracle(x, w, y, upstream=None, reduction="mean", ignore=-100):
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    z = xd @ wd.t()
    live = y != ignore
    each = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, y.clamp(min=0).unsqueeze(1)).squeeze(1), torch.zeros((), dtype=torch.float64, device=x.device))
    loss = each if reduction == "none" else each.sum() / (live.sum() if reduction == "mean" else 1)
    up = torch.ones_like(loss) if upstream is None else upstream.double()
    return (loss.detach(),) + torch.autograd.grad(loss, (xd, wd), up)


def near(got, want, tol=4e-3):
    assert torch.isfinite(got).all()
    scale = want.norm()
    assert float((got.double() - want).norm()) <= tol * float(scale) + 1e-12, (float((got.double() - want).norm()), float(scale))


def run(x, w, y, upstream=None, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, y, **kw)
    up = torch.ones_like(loss) if upstream is None else upstream
    gx, gw = torch.autograd.grad(loss, (x, w), up)
    torch.cuda.synchronize()
    assert gg.default_runtime().poll_status(True) == ""
    assert loss.dtype == torch.float32 and gx.dtype == gw.dtype == torch.bfloat16
    return loss.detach(), gx, gw


SIZES = [(1, 8, 1), (1, 64, 2), (1, 256, 1000), (3, 72, 129), (64, 256, 1000), (127, 128, 255), (128, 200, 2049), (129, 64, 300), (255, 520, 513),
         (257, 1000, 5000), (300, 2048, 10007), (1000, 136, 33000), (2049, 264, 2500), (700, 7168, 1500), (33, 640, 4000), (65, 320, 777), (224, 96, 3001), (225, 96, 3001),
         (448, 512, 1025), (449, 512, 1025), (640, 192, 70000), (1024, 64, 131073), (1025, 72, 2000),
         (192, 72, 30001), (193, 264, 2000), (384, 520, 1500), (385, 96, 3001), (530, 200, 40000), (576, 136, 2049), (577, 72, 2000)]


@pytest.mark.parametrize("T,H,V", SIZES)
def test_mean_with_ignored_tokens(native, T, H, V):
    x, w, y = make(T, H, V, seed=T)
    y[torch.rand(T, device=DEV) < 0.2] = -100
    y[0] = V - 1
    loss, gx, gw = run(x, w, y)
    want = oracle(x, w, y)
    torch.testing.assert_close(loss.double(), want[0], rtol=2e-6, atol=2e-5)
    near(gx, want[1])
    near(gw, want[2])
    assert not gx[y == -100].any()


@pytest.mark.parametrize("T,H,V", SIZES[2:])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_other_reductions(native, T, H, V, reduction):
    x, w, y = make(T, H, V, seed=T + 1)
    y[T // 2] = 0                                     # counts under ignore_index = 1
    y[T - 1] = 1
    up = torch.randn(T, device=DEV) if reduction == "none" else torch.tensor(0.37, device=DEV)
    loss, gx, gw = run(x, w, y, up, reduction=reduction, ignore_index=1)
    want = oracle(x, w, y, up, reduction, ignore=1)
    torch.testing.assert_close(loss.double(), want[0], rtol=2e-6, atol=2e-5 * (T if reduction == "sum" else 1))
    near(gx, want[1])
    near(gw, want[2])


# ------------------------------------------------------------------------------------------------------------------- edges
@pytest.mark.parametrize("T", [20, 200, 500])
def test_tokens_that_the_model_is_sure_of(native, T):
    """A target that stands out by 14 (p = 1 - 1e-4 or so): its gradient is the small number 1 - p, and keeps its digits.  p - 1 from the forward's
    fp32 logit: a few 1e-6 of a logit of 14, relative to 1 - p; then bf16 (2^-9), with the other columns' sum along W."""
    H, V = 4096, 600
    g = torch.Generator(device="cpu").manual_seed(T)
    w = torch.sign(torch.randn(V, H, generator=g)).to(torch.bfloat16).to(DEV) / 64          # |w|^2 = 1
    y = torch.randint(0, V, (T,), generator=g).to(DEV)
    x = (14.0 * w[y].float() + 0.01 * torch.randn(T, H, generator=g).to(DEV)).to(torch.bfloat16)
    loss, gx, _ = run(x, w, y, reduction="none", upstream=torch.ones(T, device=DEV))
    want = oracle(x, w, y, torch.ones(T, device=DEV), "none")
    assert float(want[0].max()) < 2e-3
    torch.testing.assert_close(loss.double(), want[0], rtol=1e-2, atol=3e-7)
    near(gx, want[1], 1e-2)


def test_a_vocabulary_of_one(native):
    x, w, y = make(50, 64, 1)
    loss, gx, gw = run(x, w, y)
    assert float(loss) == 0.0 and not gx.any() and not gw.any()


def test_gradient_against_differences(native):
    """(loss(a) - loss(b)) against the gradient half way, along random directions.  Steps of 2 % of each value: the third-order term is
    below 1 % of the difference, the losses' own errors (2e-6 of about 6) below 1 % of differences of at least 1e-2."""
    for T, H, V in ((40, 128, 300), (300, 64, 500)):
        x, w, y = make(T, H, V, seed=T)
        g = torch.Generator(device=DEV).manual_seed(3)
        for k in range(4):
            dx, dw = torch.randn(x.shape, generator=g, device=DEV) * x.abs() * 0.02, torch.randn(w.shape, generator=g, device=DEV) * w.abs() * 0.02
            if k % 2 == 0:        # along the gradient, where the difference is largest
                _, gx, gw = run(x, w, y, reduction="sum")
                dx, dw = gx.float().sign() * dx.abs(), gw.float().sign() * dw.abs()
            xa, xb, wa, wb = (x + dx).to(x.dtype), (x - dx).to(x.dtype), (w + dw).to(w.dtype), (w - dw).to(w.dtype)
            mid_x, mid_w = ((xa.float() + xb.float()) / 2).to(x.dtype), ((wa.float() + wb.float()) / 2).to(w.dtype)
            _, gx, gw = run(mid_x, mid_w, y, reduction="sum")
            with torch.no_grad():
                diff = float(linear_cross_entropy(xa, wa, y, reduction="sum").double() - linear_cross_entropy(xb, wb, y, reduction="sum").double())
            want = float((gx.double() * (xa.double() - xb.double())).sum() + (gw.double() * (wa.double() - wb.double())).sum())
            size = float((gx.double() * (xa.double() - xb.double())).norm() + (gw.double() * (wa.double() - wb.double())).norm())
            assert abs(diff - want) <= 0.02 * abs(want) + 0.05 * size + 1e-2, (T, k, diff, want, size)


@pytest.mark.parametrize("T", [20, 300])
def test_a_repeated_call_gives_the_same_bits(native, T):
    x, w, y = make(T, 512, 9000)
    a, b = run(x, w, y), run(x, w, y)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, y), a[0])


@pytest.mark.parametrize("T", [1, 33, 300, 1000])
def test_repeated_calls_of_many_units_give_the_same_bits(native, T):
    """Several units for every pair of CTAs, whichever is free first."""
    x, w, y = make(T, 264, 60001)
    load = torch.empty(64 << 20, device=DEV)
    a = run(x, w, y, reduction="none", upstream=torch.ones(T, device=DEV))
    for i in range(8):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):            # other work beside it, begun at other times
            for _ in range(i):
                load.add_(1.0)
        b = run(x, w, y, reduction="none", upstream=torch.ones(T, device=DEV))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("T", [48, 500])
def test_one_gradient_only_and_twice(native, T):
    x, w, y = make(T, 256, 3000)
    _, gx, gw = run(x, w, y)
    for which in (0, 1):
        ts = [x.detach().requires_grad_(which == 0), w.detach().requires_grad_(which == 1)]
        loss = linear_cross_entropy(ts[0], ts[1], y)
        first, = torch.autograd.grad(loss, ts[which], retain_graph=True)
        second, = torch.autograd.grad(loss, ts[which])
        assert torch.equal(first, second)
        near(first, (gx, gw)[which].double(), 1e-5 if which else 1e-2)     # (dx may be split otherwise)
    xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)      # both wanted by the graph, one by the caller
    only, = torch.autograd.grad(linear_cross_entropy(xs, ws, y), ws)
    assert torch.equal(only, gw)


def test_strides_leading_dimensions_and_alignment(native):
    T, H, V = 6 * 17, 136, 700
    x, w, y = make(T, H, V)
    want = run(x, w, y, reduction="none", upstream=torch.ones(T, device=DEV))
    wide = torch.zeros(T, 3 * H, dtype=torch.bfloat16, device=DEV)
    wide[:, H:2 * H] = x
    odd = torch.zeros(T * H + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, H).copy_(x)
    turned = w.t().contiguous().t()
    padded = torch.zeros(V, H + 8, dtype=torch.bfloat16, device=DEV)
    padded[:, :H] = w
    y2 = torch.stack([y, y], 1)[:, 0]
    for xx in (wide[:, H:2 * H], odd, x.view(6, 17, H)):
        for ww in (w, turned, padded[:, :H]):
            yy = y2.reshape(6, 17) if xx.dim() == 3 else y2
            loss, gx, gw = run(xx, ww, yy, reduction="none", upstream=torch.ones(yy.shape, device=DEV))
            assert loss.shape == yy.shape and gx.shape == xx.shape and gw.shape == ww.shape
            for got, b in zip((loss.reshape(-1), gx.reshape(T, H), gw), want):
                assert torch.equal(got, b)
    xe = x.detach().requires_grad_(True)
    linear_cross_entropy(xe, w, y, reduction="none").sum().backward()               # an expanded gradient comes back
    assert torch.equal(xe.grad, run(x, w.detach(), y, reduction="sum", upstream=torch.tensor(1.0, device=DEV))[1])


def test_nothing_and_nothing_counted(native):
    x, w, y = make(5, 64, 100)
    for reduction in ("mean", "sum", "none"):
        xe, we = x[:0].detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(xe, we, y[:0], reduction=reduction)
        gx, gw = torch.autograd.grad(loss, (xe, we), torch.ones_like(loss))
        assert loss.shape == (torch.Size([0]) if reduction == "none" else torch.Size([])) and gx.shape == (0, 64) and not gw.any()
        if reduction != "none":
            assert torch.isnan(loss) if reduction == "mean" else float(loss.detach()) == 0.0
    for T in (5, 300):
        x, w, y = make(T, 64, 100)
        xe, we = x.requires_grad_(True), w.requires_grad_(True)
        loss = linear_cross_entropy(xe, we, torch.full_like(y, -100))
        gx, gw = torch.autograd.grad(loss, (xe, we))
        assert torch.isnan(loss) and not gx.any() and not gw.any()


@pytest.mark.parametrize("T", [30, 400, 700])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_rows_of_ignored_tokens(native, T, bad):
    """An ignored token's hidden state may hold anything: the losses and the other tokens' gradients do not see it."""
    x, w, y = make(T, 128, 1000)
    clean = run(x, w.detach(), torch.where(torch.arange(T, device=DEV) % 7 == 3, -100, y))
    dirty = x.detach().clone()
    dirty[3::7] = bad
    y[3::7] = -100
    xe = dirty.requires_grad_(True)
    loss = linear_cross_entropy(xe, w.detach(), y)
    gx, = torch.autograd.grad(loss, xe)
    assert torch.equal(loss, clean[0]) and torch.equal(gx, clean[1]) and not gx[3::7].any()


@pytest.mark.parametrize("T", [30, 400, 700])
def test_columns_that_are_out_of_reach(native, T):
    """Logits of -inf and of the type's lowest values among the others (masked vocabulary): probability zero, no NaN."""
    x, w, y = make(T, 64, 1000)
    x = x.clone()
    x[:, 0] = 1.0
    w = w.clone()
    w[500:700] = 0
    w[500:600, 0] = -float("inf")
    w[600:700, 0] = torch.finfo(torch.bfloat16).min
    y = torch.where((y >= 500) & (y < 700), 0, y)
    with torch.no_grad():
        loss = linear_cross_entropy(x, w, y, reduction="none")
    keep = torch.cat([w[:500], w[700:]])
    z = x.double() @ keep.double().t()
    want = torch.logsumexp(z, 1) - (x.double() * w[y].double()).sum(1)
    torch.testing.assert_close(loss.double(), want, rtol=2e-6, atol=2e-5)
    w[500:600, 0] = torch.finfo(torch.bfloat16).min
    xe, we = x.requires_grad_(True), w.requires_grad_(True)
    gx, gw = torch.autograd.grad(linear_cross_entropy(xe, we, y), (xe, we))
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all() and not gw[500:700].any()


@pytest.mark.parametrize("T", [30, 400, 700])
def test_rows_at_the_lowest_value(native, T):
    """Every logit at the type's lowest value: all columns alike, loss ln(V), a gradient of p = 1 / V."""
    V = 1000
    x, w = torch.zeros(T, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(V, 64, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 1.0
    w[:, 0] = torch.finfo(torch.bfloat16).min
    x[:, 1] = 0.5
    y = torch.randint(0, V, (T,), device=DEV)
    loss, gx, gw = run(x, w, y, reduction="none", upstream=torch.ones(T, device=DEV))
    torch.testing.assert_close(loss.double(), torch.full((T,), float(V), dtype=torch.float64, device=DEV).log(), rtol=1e-6, atol=0)
    want = torch.full((V, T), 1.0 / V, dtype=torch.float64, device=DEV)
    want[y, torch.arange(T, device=DEV)] -= 1.0
    near(gw, want @ x.double())


@pytest.mark.parametrize("T", [30, 400, 700])
def test_target_outside_the_vocabulary(native, T):
    from streamep_b200 import LocalWorld
    buf = LocalWorld(1, arena_bytes=64 << 20).buffers[0]
    x, w, y = make(T, 64, 1000)
    for bad in (1000, -1, 1 << 40):
        y2 = y.clone()
        y2[T // 2] = bad
        xe, we = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(xe, we, y2, buffer=buf)
        gx, gw = torch.autograd.grad(loss, (xe, we))
        assert torch.isnan(loss) and torch.isnan(gx[T // 2]).all() and torch.isfinite(gx[:T // 2]).all()
        with pytest.raises(StreamEPError, match="outside the vocabulary"):
            buf.check_status()
    assert torch.isfinite(linear_cross_entropy(x, w, y, buffer=buf))
    buf.check_status()


def test_streams_and_capture(native):
    x, w, y = make(200, 256, 5000)
    want = run(x, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        xe, we = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(xe, we, y)
    got = torch.autograd.grad(loss, (xe, we))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])
    xs, ws = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(xs, ws, y)
        grads = torch.autograd.grad(loss, (xs, ws))
    for scale in (1.0, 0.5, 1.0):
        with torch.no_grad():
            xs.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(grads[0], want[1]) and torch.equal(grads[1], want[2])


@pytest.mark.parametrize("shape", [(48, 256, 5000), (700, 512, 3000)])
def test_backward_captured_on_its_own(native, shape):
    """A graph with the backward alone may be replayed more than once after one forward."""
    x, w, y = make(*shape)
    want = run(x, w, y)
    xs, ws = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    up = torch.ones((), device=x.device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = linear_cross_entropy(xs, ws, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = torch.autograd.grad(loss, (xs, ws), up)
    for scale in (1.0, 0.5, 1.0):
        up.fill_(scale)
        graph.replay()
        torch.cuda.synchronize()
        for got, g in zip(grads, want[1:]):
            assert torch.equal(got, g * scale)       # (a power of two)


def test_forward_and_backward_captured_apart(native):
    x, w, y = make(300, 256, 5000)
    want = run(x, w, y)
    xs, ws = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(first, stream=side):
        loss = linear_cross_entropy(xs, ws, y)
    with torch.cuda.graph(second, pool=first.pool(), stream=side):
        grads = torch.autograd.grad(loss, (xs, ws))
    for graph in (first, second, second, first, first, second):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(grads[0], want[1]) and torch.equal(grads[1], want[2])


def test_two_streams_at_once(native):
    """Both calls want every SM: neither may wait for the other's blocks."""
    xs = [make(1500, 512, 20000, seed=s) for s in (1, 2)]
    want = [run(*a) for a in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    out = []
    for _ in range(3):
        out = []
        for s, (x, w, y) in zip(streams, xs):
            with torch.cuda.stream(s):
                xe, we = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
                loss = linear_cross_entropy(xe, we, y)
                out.append((loss,) + torch.autograd.grad(loss, (xe, we)))
    torch.cuda.synchronize()
    assert gg.default_runtime().poll_status(True) == ""
    for got, b in zip(out, want):
        assert all(torch.equal(p, q) for p, q in zip(got, b))


def test_offsets_beyond_32_bits(native):
    """A projection of 2.3 G elements, and hidden states of 2.4 G."""
    g = torch.Generator(device=DEV).manual_seed(0)
    for T, H, V in ((2, 16384, 140_000), (300_000, 8192, 300)):
        x = torch.empty(T, H, dtype=torch.bfloat16, device=DEV).normal_(0, 0.1, generator=g).requires_grad_(True)
        w = torch.empty(V, H, dtype=torch.bfloat16, device=DEV).normal_(0, 0.02, generator=g).requires_grad_(True)
        y = torch.randint(0, V, (T,), generator=g, device=DEV)
        y[-1] = V - 1
        loss = linear_cross_entropy(x, w, y, reduction="none")
        gx, gw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        rows = torch.tensor([0, T - 1], device=DEV)
        with torch.no_grad():
            z = torch.cat([x[rows].double() @ w[a:a + 5000].double().t() for a in range(0, V, 5000)], 1)
            lse = torch.logsumexp(z, 1, keepdim=True)
            torch.testing.assert_close(loss[rows].double(), (lse - z.gather(1, y[rows, None])).squeeze(1), rtol=2e-6, atol=2e-5)
            dz = (z - lse).exp()
            dz[torch.arange(2, device=DEV), y[rows]] -= 1.0
            near(gx[rows], sum(dz[:, a:a + 5000] @ w[a:a + 5000].double() for a in range(0, V, 5000)))
            if T == 2:
                near(gw[-1000:], dz[:, -1000:].t() @ x.double())
        del x, w, loss, gx, gw, z
        torch.cuda.empty_cache()


def test_refusals(native):
    x, w, y = make(8, 64, 100)
    for args, kw in (((x.float(), w, y), {}), ((x, w.float(), y), {}), ((x, w, y.int()), {}), ((x[:, :60], w[:, :60], y), {}), ((x, w[:, :56], y), {}),
                     ((x, w, y[:-1]), {}), ((x, w[:0], y), {}), ((x.cpu(), w, y), {}), ((x, w.cpu(), y), {}), ((x, w, y.cpu()), {}),
                     ((x, w, y), dict(reduction="max")), ((x, w[0], y), {}), ((x, w, y.view(2, 4)), {})):
        with pytest.raises(ValueError):
            linear_cross_entropy(*args, **kw)
    xe = x.detach().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):      # (the autograd engine turns every exception into this type)
        torch.autograd.grad(linear_cross_entropy(xe, w, y), xe, create_graph=True)
    xe = x.detach().requires_grad_(True)
    loss = linear_cross_entropy(xe, w, y)
    w.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(loss, xe)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        linear_cross_entropy(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w, y)
    from streamep_b200 import LocalWorld
    buf = LocalWorld(1, arena_bytes=64 << 20).buffers[0]
    buf.runtime.destroy()
    with pytest.raises(ValueError, match="destroyed"):
        linear_cross_entropy(x, w, y, buffer=buf)
