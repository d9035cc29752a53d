"""grad_norm, clip_grad_norm_ and adamw_step_ against 64-bit arithmetic: types, lengths around vectors and chunks, places off every
boundary, long lists, strides, non-finite values, refusals.

Tolerances.  Norm: a square is rounded once (2^-24), a thread adds at most about 70 of them in fp32 here (70 x 2^-24, halved by the root),
doubles from there: 3e-6.  Scaling: that, the factor's and the product's rounding: 4e-6 on fp32; bf16 results within one more
rounding (2^-8 of the value).  AdamW: each of m, v, w is a handful of fp32 operations on terms that may cancel: 1e-6 of the sum of their magnitudes."""
import math

import pytest
import torch

from streamep_b200.ops import adamw_step_, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def views(sizes, dtypes, packed, seed=0, std=1.0, gap=0):
    """Tensors of the given lengths, each in memory of its own or end to end behind `gap` elements."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    flats = {d: torch.zeros(gap + sum(sizes) + 1, dtype=d, device=DEV) for d in set(dtypes)}
    at = {d: gap for d in flats}
    for n, d in zip(sizes, dtypes):
        if packed:
            t = flats[d][at[d]:at[d] + n]
            at[d] += n
        else:
            t = torch.empty(n, dtype=d, device=DEV)
        out.append(t.normal_(0.0, std, generator=g))
    return out


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


LISTS = [([1], False), ([0], False), ([7], True), ([8, 0, 1, 4095, 4096, 4097], True), ([3, 1023, 1024, 1025, 2, 2047, 100_003], True),
         ([3, 1023, 1024, 1025, 2, 2047, 100_003], False), ([5] * 1500, True), ([1000 + i for i in range(1100)], True), ([3_000_001, 17, 5_000_000], True)]


@pytest.mark.parametrize("dtypes", [(BF,), (F32,), (BF, F32, BF)])
@pytest.mark.parametrize("case", range(len(LISTS)))
def test_norm_and_clip(native, case, dtypes):
    sizes, packed = LISTS[case]
    kinds = [dtypes[i % len(dtypes)] for i in range(len(sizes))]
    for gap in ((0, 1, 3) if packed else (0,)):
        ts = views(sizes, kinds, packed, seed=case, gap=gap)
        before = [t.clone() for t in ts]
        want = norm64(ts)
        got = grad_norm(ts)
        assert got.dtype == F32 and got.shape == () and got.is_cuda
        assert abs(float(got) - want) <= 3e-6 * want
        again = clip_grad_norm_(ts, want * 2 + 1)                  # below the limit: nothing changes
        assert torch.equal(again, got) and all(torch.equal(a, b) for a, b in zip(ts, before))
        limit = want * 0.37
        again = clip_grad_norm_(ts, limit)
        assert torch.equal(again, got)
        f = limit / (want + 1e-6)
        for t, b in zip(ts, before):
            torch.testing.assert_close(t.double(), b.double() * f, rtol=4e-6 + (2 ** -8 if t.dtype == BF else 0), atol=1e-30)


def test_empty_lists(native):
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    empty = torch.empty(0, device=DEV)
    assert float(clip_grad_norm_([empty, empty], 1.0)) == 0.0
    zero = torch.zeros(100, device=DEV)
    assert float(clip_grad_norm_([zero], 0.0)) == 0.0 and not zero.any()


def test_neighbours_of_packed_tensors_stay(native):
    flat = torch.ones(1000, dtype=BF, device=DEV)
    ts = [flat[3:250], flat[251:500], flat[777:778]]
    clip_grad_norm_(ts, 0.5)
    mask = torch.zeros(1000, dtype=torch.bool, device=DEV)
    mask[3:250] = mask[251:500] = mask[777:778] = True
    assert (flat[~mask] == 1).all() and (flat[mask] < 0.1).all()


def test_strided(native):
    base = torch.randn(64, 48, device=DEV)
    t, gaps = base.clone().t(), torch.randn(40, 30, device=DEV)[:, 3:20]
    want_t, want_g = t.clone(), gaps.clone()
    want = norm64([t, gaps])
    assert abs(float(grad_norm([t, gaps])) - want) <= 3e-6 * want
    wide = torch.randn(1, 5, device=DEV).expand(7, 5)
    assert abs(float(grad_norm([wide])) - norm64([wide])) <= 3e-6 * norm64([wide])
    version = gaps._version
    clip_grad_norm_([t, gaps], 1.0)
    assert gaps._version > version
    for got, b in ((t, want_t), (gaps, want_g)):
        torch.testing.assert_close(got.double(), b.double() / (want + 1e-6), rtol=4e-6, atol=1e-30)


@pytest.mark.parametrize("bad,factor", [(float("nan"), float("nan")), (float("inf"), 0.0), (-float("inf"), 0.0)])
def test_non_finite(native, bad, factor):
    a, b = torch.ones(5000, device=DEV), torch.ones(300, dtype=BF, device=DEV)
    a[4321] = bad
    norm = clip_grad_norm_([a, b], 1.0)
    assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
    assert torch.isnan(a[4321])
    for t in (a[:4000], b):
        assert torch.isnan(t).all() if math.isnan(factor) else (t == 0).all()


def test_versions_and_streams(native):
    t = torch.ones(1 << 20, device=DEV)
    version = t._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t.mul_(2.0)
        norm = clip_grad_norm_([t], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert t._version > version + 1 and float(norm) == 2048.0
    torch.testing.assert_close(t, torch.full_like(t, 2.0 / 2048.0), rtol=1e-6, atol=0)


def test_captured(native):
    t = [torch.randn(5000, device=DEV), torch.randn(777, dtype=BF, device=DEV)]
    grad_norm(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = grad_norm(t)
    t[0].mul_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert abs(float(norm) - norm64(t)) <= 3e-6 * norm64(t)


def test_refusals(native):
    t = torch.randn(100, device=DEV)
    with pytest.raises(ValueError):
        clip_grad_norm_([t, t], 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_([t[:60], t[50:]], 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_([t], -1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_([t], float("nan"))
    with pytest.raises(ValueError):
        clip_grad_norm_([t[:1].expand(5)], 1.0)
    for bad in (torch.randn(5), torch.randn(5, device=DEV, dtype=torch.float64), torch.arange(5, device=DEV)):
        with pytest.raises(ValueError):
            grad_norm([t, bad])
    p, m, v = torch.randn(100, device=DEV), torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    ok = dict(step=1, lr=0.1)
    for change in (dict(step=0), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(max_norm=1.0), dict(skip_nonfinite=True), dict(masters=[]), dict(masters=[m.to(BF)]),
                   dict(norm=torch.ones((), device=DEV), max_norm=-2.0), dict(norm=torch.ones(2, device=DEV), max_norm=1.0)):
        with pytest.raises(ValueError):
            adamw_step_([p], [t], [m], [v], **{**ok, **change})
    for lists in (([p], [t[:50]], [m], [v]), ([p], [t], [m], []), ([p, p], [t, t], [m, m.clone()], [v, v.clone()]), ([p.double()], [t], [m], [v]),
                  ([p], [t], [m], [m]), ([p], [t], [p], [v]), ([p], [t], [m.to(BF)], [v]), ([p[::2]], [t[::2]], [m[::2]], [v[::2]])):
        with pytest.raises(ValueError):
            adamw_step_(*lists, **ok)


def oracle(p, g, m, v, w, o, f):
    p, g, m, v = p.double(), g.double() * f, m.double(), v.double()
    w = p if w is None else w.double()
    b1, b2 = o["betas"]
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    move = o["lr"] * (m2 / (1 - b1 ** o["step"])) / ((v2 / (1 - b2 ** o["step"])).sqrt() + o["eps"])
    scale = o["lr"] * ((b1 * m.abs() + (1 - b1) * g.abs()) / (1 - b1 ** o["step"])) / ((v2 / (1 - b2 ** o["step"])).sqrt() + o["eps"])
    return m2, b1 * m.abs() + (1 - b1) * g.abs(), v2, w * (1 - o["lr"] * o["weight_decay"]) - move, w.abs() + scale


ADAM_SIZES = [[1], [0, 5], [4, 3, 1, 4095, 4096, 4097, 30_001], [7] * 700, [2_000_003, 11], [5_000_003, 2, 4_000_001, 2047]]


@pytest.mark.parametrize("kind", ["master", "bf16", "fp32", "fp32 bf16 grads"])
@pytest.mark.parametrize("case", range(len(ADAM_SIZES)))
def test_adamw(native, case, kind):
    sizes = ADAM_SIZES[case]
    n = len(sizes)
    pt, gt = {"master": (BF, BF), "bf16": (BF, BF), "fp32": (F32, F32), "fp32 bf16 grads": (F32, BF)}[kind]
    for packed, gap in ((False, 0), (True, 0), (True, 1), (True, 6)):
        ps, gs = views(sizes, [pt] * n, packed, 1, 0.5, gap), views(sizes, [gt] * n, packed, 2, 0.1, gap)
        # (places that do not go together: the moments stand elsewhere)
        ms, vs = views(sizes, [F32] * n, packed, 3, 0.1, gap if case != 2 else 2), views(sizes, [F32] * n, packed, 4, 0.1, gap)
        for v in vs:
            v.square_()
        ws = [p.float() + 1e-4 for p in ps] if kind == "master" else None
        o = dict(step=3, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
        norm = grad_norm(gs)
        limit = 0.25 * norm64(gs)
        f = min(1.0, limit / (norm64(gs) + 1e-6))
        want = [oracle(p, g, m, v, w, o, f) for p, g, m, v, w in zip(ps, gs, ms, vs, ws or [None] * n)]
        kept = [g.clone() for g in gs]
        versions = [p._version for p in ps]
        adamw_step_(ps, gs, ms, vs, masters=ws, norm=norm, max_norm=limit, **o)
        assert all(torch.equal(a, b) for a, b in zip(gs, kept)) and all(p._version > v for p, v in zip(ps, versions))
        for i in range(n):
            m2, m_size, v2, w2, w_size = want[i]
            assert ((ms[i].double() - m2).abs() <= 4e-6 * m_size + 1e-30).all()     # (the factor's error included)
            assert ((vs[i].double() - v2).abs() <= 1e-5 * v2 + 1e-30).all()
            if ws is not None:
                assert ((ws[i].double() - w2).abs() <= 1e-5 * w_size).all()
                assert torch.equal(ps[i], ws[i].to(BF))
            else:
                assert ((ps[i].double() - w2).abs() <= 1e-5 * w_size + (2 ** -8 * w2.abs() if pt == BF else 0)).all()


def test_adamw_without_clipping_and_skipped(native):
    p, g, m, v = (torch.randn(1000, device=DEV) for _ in range(4))
    v.abs_()
    o = dict(step=1, lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    m2, m_size, v2, w2, w_size = oracle(p, g, m, v, None, o, 1.0)
    q, a, b = p.clone(), m.clone(), v.clone()
    adamw_step_([q], [g], [a], [b], **o)
    assert ((a.double() - m2).abs() <= 1e-6 * m_size).all() and ((q.double() - w2).abs() <= 1e-5 * w_size).all()
    g[17] = float("inf")
    keep = [t.clone() for t in (q, a, b)]
    adamw_step_([q], [g], [a], [b], norm=grad_norm([g]), max_norm=1.0, skip_nonfinite=True, **o)
    assert all(torch.equal(x, y) for x, y in zip((q, a, b), keep))
    adamw_step_([q], [g], [a], [b], norm=grad_norm([g]), max_norm=1.0, **o)
    assert torch.isnan(q[17]) and torch.isfinite(q[18:]).all()


def test_adamw_gradient_in_another_layout(native):
    p = torch.randn(30, 50, device=DEV)
    g = torch.randn(50, 30, device=DEV).t()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    o = dict(step=1, lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    w2, w_size = oracle(p, g, m, v, None, o, 1.0)[3:]
    adamw_step_([p], [g], [m], [v], **o)
    assert ((p.double() - w2).abs() <= 1e-5 * w_size).all()
