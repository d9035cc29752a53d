"""gated_scan and gated_scan_step_ against 64-bit arithmetic: lengths around chunks and groups of chunks, packed sequences (empty ones, single
rows, rows that belong to none), states, strides, odd channels, non-finite values, streams, captured graphs, bad offsets, refusals.

Tolerances, in units of 2^-24.  A sigmoid is off by 8 of itself (exponential 4, sum, reciprocal 2, difference to 1), and |gate| more where the
exponent is rounded once (bf16).  A row's contribution passes, on its way to a later one, one product by a keep (its error, a rounding, and a
rounding where products are joined) and one sum a row: with m the recurrence of |x| and r that of m, h is off by K r, K = 12 + |gate|.
The backward is the same recurrence of |dh|, the gradients one product and one difference more.  What is returned in fewer bits is rounded once."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.errors import StreamEPError
from streamep_b200.ops import gated_scan, gated_scan_step_

gpu = pytest.mark.gpu
DEV = "cuda"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
ULP = 2.0 ** -24


def recur(a, b):
    """y_t = a_t y_{t-1} + b_t along the first dimension, from zero."""
    step = 1
    while step < len(a):
        b = torch.cat([b[:step], a[step:] * b[:-step] + b[step:]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def test_the_oracle():
    g = torch.Generator().manual_seed(0)
    a, b = torch.rand(37, 5, generator=g, dtype=F64), torch.randn(37, 5, generator=g, dtype=F64)
    y, rows = torch.zeros(5, dtype=F64), []
    for t in range(37):
        y = a[t] * y + b[t]
        rows.append(y)
    torch.testing.assert_close(recur(a, b), torch.stack(rows), rtol=1e-13, atol=1e-13)


def oracle(x, gate, initial, spans, dh=None, dfinal=None, h_rounded=None):
    """Per quantity the value and the bound without the result's own rounding; rows of no sequence are zero."""
    N, D = x.shape
    K = (12 + (float(gate.abs().nan_to_num(0, 0, 0).max()) if x.dtype == BF and N else 0.0)) * ULP
    x, gate = x.double(), gate.double()
    S = len(spans)
    first = initial.double() if initial is not None else torch.zeros(S, D, dtype=F64, device=x.device)
    zeros = lambda n: torch.zeros(n, D, dtype=F64, device=x.device)
    out = {k: [zeros(n), zeros(n)] for k, n in (("h", N), ("final", S), ("dx", N), ("dgate", N), ("dinitial", S))}
    for s, (p, q) in enumerate(spans):
        out["final"][0][s] = first[s]
        last = dfinal.double()[s] if dfinal is not None else torch.zeros(D, dtype=F64, device=x.device)
        out["dinitial"][0][s] = last
        if p == q:
            continue
        keep, take = torch.sigmoid(gate[p:q]), torch.sigmoid(-gate[p:q])
        follow = lambda start, v: recur(keep, torch.cat([v[:1] + keep[:1] * start, v[1:]]))
        h = follow(first[s], take * x[p:q])
        m = follow(first[s].abs(), take * x[p:q].abs())
        r = follow(torch.zeros_like(first[s]), m)
        out["h"][0][p:q], out["h"][1][p:q] = h, K * r
        out["final"][0][s], out["final"][1][s] = h[-1], K * r[-1]
        if dh is None and dfinal is None:
            continue
        up = dh[p:q].double() if dh is not None else zeros(q - p)
        back = torch.cat([keep[1:], zeros(1)]).flip(0)           # a row's gradient is weighted with the keep of the row behind it
        end = torch.cat([zeros(q - p - 1), last[None]])
        g = recur(back, (up + end).flip(0)).flip(0)
        mg = recur(back, (up.abs() + end.abs()).flip(0)).flip(0)
        rg = recur(back, mg.flip(0)).flip(0)
        before = torch.cat([first[s][None], (h_rounded[p:q].double() if h_rounded is not None else h)[:-1]])
        out["dx"][0][p:q], out["dx"][1][p:q] = take * g, K * take * (rg + mg)
        slope = keep * take
        out["dgate"][0][p:q] = g * slope * (before - x[p:q])
        out["dgate"][1][p:q] = K * slope * ((before - x[p:q]).abs() * (rg + 2 * mg) + mg * (before.abs() + x[p:q].abs()))
        out["dinitial"][0][s], out["dinitial"][1][s] = keep[0] * g[0], K * keep[0] * (rg[0] + mg[0])
    return out


def near(got, want, what):
    value, slack = want
    got = got.reshape(value.shape)
    half = torch.finfo(got.dtype).eps / 2
    over = (got.double() - value).abs() - (slack + half * value.abs())
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3e} above the bound at {int(over.argmax())}"


def inputs(N, D, dtype, seed=0, joint=False, off=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    centre = torch.empty(D, device=DEV).uniform_(-2.0, 9.0, generator=g)
    x = torch.randn(N, D, generator=g, device=DEV)
    gate = torch.randn(N, D, generator=g, device=DEV) + centre
    if joint:
        both = torch.cat([x, gate], 1).to(dtype)
        return both[:, :D], both[:, D:], torch.randn(N, D, generator=g, device=DEV).to(dtype)
    if off:
        flat = torch.zeros(N * D + off, device=DEV, dtype=dtype)
        flat[off:] = x.to(dtype).view(-1)
        return flat[off:].view(N, D), gate.to(dtype), torch.randn(N, D, generator=g, device=DEV).to(dtype)
    return x.to(dtype), gate.to(dtype), torch.randn(N, D, generator=g, device=DEV).to(dtype)


def check(x, gate, dh, spans, shape=None, offsets=None, initial=None, dfinal=None, train=True):
    """One call on rows x, gate (viewed as `shape`) and its gradients."""
    N, D = x.shape
    shape = shape or (N, D)
    leaves = [t.detach().requires_grad_(train) for t in (x.view(shape), gate.view(shape))]
    if initial is not None:
        leaves.append(initial.detach().requires_grad_(train))
    h, final = gated_scan(leaves[0], leaves[1], initial_state=leaves[2] if initial is not None else None, offsets=offsets, return_state=True)
    assert h.shape == shape and h.dtype == x.dtype and final.shape == (len(spans), D) and final.dtype == F32
    want = oracle(x, gate, initial, spans, dh if train else None, dfinal, h.detach().reshape(N, D))
    near(h.detach(), want["h"], "h")
    near(final.detach(), want["final"], "final")
    if not train:
        return [h, final]
    outs, ups = ([h, final], [dh.view(shape), dfinal]) if dfinal is not None else ([h], [dh.view(shape)])
    grads = torch.autograd.grad(outs, leaves, ups)
    for n, g in zip(("dx", "dgate", "dinitial"), grads):
        near(g, want[n], n)
    ops.check_status()
    return [h.detach(), final.detach(), *grads]


def dense(B, T, D, dtype, state=True, **kw):
    x, gate, dh = inputs(B * T, D, dtype, seed=B * 131 + T * 7 + D, **kw)
    g = torch.Generator(device=DEV).manual_seed(9)
    initial, dfinal = (torch.randn(B, D, generator=g, device=DEV) for _ in range(2)) if state else (None, None)
    return check(x, gate, dh, [(b * T, (b + 1) * T) for b in range(B)], (B, T, D), None, initial, dfinal)


DENSE = [(1, 1, 8), (3, 1, 64), (2, 5, 7), (1, 31, 64), (1, 127, 64), (1, 128, 64), (1, 129, 64), (4, 128, 72), (5, 64, 200), (2, 300, 136), (3, 255, 1001),
         (2, 513, 33), (1, 4097, 64), (1, 9000, 24), (700, 3, 5), (1, 20000, 40), (2, 8192, 66), (1, 257, 4099)]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,D", DENSE)
def test_dense(native, B, T, D, dtype):
    dense(B, T, D, dtype)
    dense(B, T, D, dtype, state=False)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_places(native, dtype):
    for D in (64, 100, 7):
        dense(3, 200, D, dtype, joint=True)
        dense(2, 150, D, dtype, off=1)
    # time before batch: no common distance between rows, so copied
    x, gate, dh = inputs(60, 16, dtype, seed=2)
    a, b = (t.view(20, 3, 16).transpose(0, 1) for t in (x, gate))
    got = gated_scan(a, b)
    assert torch.equal(got, gated_scan(a.contiguous(), b.contiguous()))
    leaf = a.detach().requires_grad_(True)
    up = torch.randn(16, 3, 20, device=DEV).to(dtype).permute(1, 2, 0)
    gl, = torch.autograd.grad(gated_scan(leaf, b), leaf, up)
    lc = a.contiguous().requires_grad_(True)
    gc, = torch.autograd.grad(gated_scan(lc, b.contiguous()), lc, up.contiguous())
    assert torch.equal(gl, gc)


PACKED = [([5], 0, 0), ([0, 0, 0], 0, 3), ([1, 0, 127, 1, 128, 0, 300, 2], 0, 0), ([130, 4096, 1, 4500, 0, 77], 7, 200), ([3] * 200, 1, 9), ([0, 9000, 0], 128, 128),
          ([17, 0, 240], 129, 300)]


@gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 37), (F32, 100), (F32, 9)])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed(native, case, dtype, D, wide):
    lengths, lead, tail = PACKED[case]
    at = [lead]
    for n in lengths:
        at.append(at[-1] + n)
    N = at[-1] + tail
    x, gate, dh = inputs(N, D, dtype, seed=case)
    outside = torch.ones(N, dtype=torch.bool, device=DEV)
    outside[at[0]:at[-1]] = False
    for t in (x, gate, dh):                              # rows of no sequence are not looked at
        t[outside] = float("nan")
    offsets = torch.tensor(at, dtype=torch.int64 if wide else torch.int32, device=DEV)
    spans = list(zip(at[:-1], at[1:]))
    g = torch.Generator(device=DEV).manual_seed(4)
    initial, dfinal = (torch.randn(len(spans), D, generator=g, device=DEV) for _ in range(2))
    clean = lambda t: torch.where(outside[:, None], torch.zeros_like(t), t)
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, initial)]
    h, final = gated_scan(*leaves[:2], initial_state=leaves[2], offsets=offsets, return_state=True)
    grads = torch.autograd.grad([h, final], leaves, [dh, dfinal])
    want = oracle(clean(x), clean(gate), initial, spans, clean(dh), dfinal, h.detach())
    for n, got in zip(("h", "final", "dx", "dgate", "dinitial"), (h.detach(), final.detach(), *grads)):
        near(got, want[n], n)
    ops.check_status()


@gpu
def test_without_rows_or_sequences(native):
    for dtype in (BF, F32):
        e = torch.empty(3, 0, 8, device=DEV, dtype=dtype)
        s = torch.randn(3, 8, device=DEV, requires_grad=True)
        h, final = gated_scan(e, e, initial_state=s, return_state=True)
        assert h.shape == (3, 0, 8) and torch.equal(final, s)
        up = torch.randn(3, 8, device=DEV)
        assert torch.equal(torch.autograd.grad(final, s, up)[0], up)
        x = torch.full((5, 8), float("nan"), device=DEV, dtype=dtype, requires_grad=True)
        h, final = gated_scan(x, x, offsets=torch.zeros(1, dtype=torch.int32, device=DEV), return_state=True)
        assert torch.equal(h, torch.zeros_like(h)) and final.shape == (0, 8)
        assert torch.equal(torch.autograd.grad(h, x, torch.ones_like(h))[0], torch.zeros_like(h))
        h = gated_scan(torch.empty(0, 4, 8, device=DEV, dtype=dtype), torch.empty(0, 4, 8, device=DEV, dtype=dtype))
        assert h.shape == (0, 4, 8)


@gpu
@pytest.mark.parametrize("D", [64, 9])
def test_subsets_of_gradients(native, D):
    x, gate, dh = inputs(600, D, F32, seed=6)
    g = torch.Generator(device=DEV).manual_seed(5)
    initial, dfinal = (torch.randn(2, D, generator=g, device=DEV) for _ in range(2))
    t = [x.view(2, 300, D), gate.view(2, 300, D), initial]
    up = dh.view(2, 300, D)

    def grads(mask, outs):
        leaves = [v.detach().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate(t)]
        h, final = gated_scan(leaves[0], leaves[1], initial_state=leaves[2], return_state=True)
        pick = [i for i in range(3) if mask >> i & 1]
        chosen = [(h, up), (final, dfinal)] if outs == 2 else [(h, up)] if outs == 0 else [(final, dfinal)]
        got = torch.autograd.grad([c[0] for c in chosen], [leaves[i] for i in pick], [c[1] for c in chosen])
        return dict(zip(pick, got))
    for outs in range(3):
        want = grads(7, outs)
        for mask in range(1, 7):
            for i, got in grads(mask, outs).items():
                assert torch.equal(got, want[i]), (outs, mask, i)
    a, b = grads(7, 0), grads(7, 1)
    both = grads(7, 2)
    for i in range(3):
        torch.testing.assert_close(a[i] + b[i], both[i], rtol=1e-4, atol=1e-4)


@gpu
def test_against_differences(native):
    B, T, D = 2, 150, 12
    x, gate, dh = inputs(B * T, D, F32, seed=8)
    g = torch.Generator(device=DEV).manual_seed(3)
    initial, dfinal = (torch.randn(B, D, generator=g, device=DEV) for _ in range(2))
    t = [x.view(B, T, D), gate.view(B, T, D), initial]
    leaves = [v.detach().requires_grad_(True) for v in t]
    h, final = gated_scan(leaves[0], leaves[1], initial_state=leaves[2], return_state=True)
    grads = torch.autograd.grad([h, final], leaves, [dh.view(B, T, D), dfinal])
    spans = [(b * T, (b + 1) * T) for b in range(B)]

    def value(parts, exact):
        if exact:
            o = oracle(parts[0].reshape(-1, D), parts[1].reshape(-1, D), parts[2], spans)
            return float((o["h"][0] * dh.double()).sum() + (o["final"][0] * dfinal.double()).sum()), \
                float((o["h"][1] * dh.double().abs()).sum() + (o["final"][1] * dfinal.double().abs()).sum()) + ULP * float((o["h"][0] * dh.double()).abs().sum())
        hh, ff = gated_scan(parts[0], parts[1], initial_state=parts[2], return_state=True)
        return float((hh.double() * dh.view(B, T, D).double()).sum() + (ff.double() * dfinal.double()).sum()), 0.0
    for i in range(3):
        v = torch.randn(t[i].shape, generator=g, device=DEV)
        step = 2.0 ** -8
        at = lambda f: [q + (f * step * v if k == i else 0.0) for k, q in enumerate(t)]
        slope = float((grads[i].double() * v.double()).sum())
        (up, e1), (down, e2) = value(at(1), True), value(at(-1), True)
        mine = (value(at(1), False)[0] - value(at(-1), False)[0]) / (2 * step)
        exact = (up - down) / (2 * step)
        rounding = (e1 + e2) / (2 * step)
        assert abs(mine - exact) <= rounding
        # the differences' own error, step^2 / 6 of a third derivative: from twice the step
        (up2, _), (down2, _) = value(at(2), True), value(at(-2), True)
        curve = abs((up2 - down2) / (4 * step) - exact)
        assert abs(slope - exact) <= curve + rounding


@gpu
@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 9)])
def test_non_finite_values_stay_in_their_sequence_and_channel(native, dtype, D):
    lengths = [100, 300, 5, 9000]
    at = [0, 100, 400, 405, 9405]
    x, gate, dh = inputs(9405, D, dtype, seed=12)
    offsets = torch.tensor(at, dtype=torch.int32, device=DEV)
    initial = torch.randn(4, D, device=DEV)

    def run(x, gate, initial, dh):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gate, initial)]
        h, final = gated_scan(*leaves[:2], initial_state=leaves[2], offsets=offsets, return_state=True)
        return [h.detach(), final.detach(), *torch.autograd.grad(h, leaves, dh)]
    want = run(x, gate, initial, dh)
    seq = torch.repeat_interleave(torch.arange(4, device=DEV), torch.tensor(lengths, device=DEV))
    for bad in (float("nan"), float("inf")):
        for s, which in ((1, 0), (1, 1), (3, 0), (0, 2), (2, 3)):
            t = [v.clone() for v in (x, gate, initial, dh)]
            t[which][s if which == 2 else at[s] + lengths[s] // 2, 3] = bad
            got = run(*t)
            for n, (a, b) in enumerate(zip(got, want)):
                same = torch.ones_like(a, dtype=torch.bool)
                rows = torch.arange(4, device=DEV) == s if n in (1, 4) else seq == s
                same[rows, 3] = False
                assert torch.equal(a[same], b[same]), (bad, s, which, n)
    # a gate of plus or minus infinity holds or replaces the state
    for sign in (1, -1):
        shut = torch.full((1, 40, D), sign * float("inf"), device=DEV, dtype=dtype)
        rows = torch.randn(1, 40, D, device=DEV).to(dtype)
        h, final = gated_scan(rows, shut, initial_state=initial[:1], return_state=True)
        assert torch.equal(h, initial[:1].to(dtype).expand(1, 40, D) if sign > 0 else rows)
        assert torch.equal(final, initial[:1] if sign > 0 else rows[:, -1].float())


@gpu
@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 9), (F32, 2000)])
def test_steps_continue_a_sequence(native, dtype, D):
    B, T = 5, 200
    x, gate, dh = inputs(B * T, D, dtype, seed=21)
    x, gate = x.view(B, T, D), gate.view(B, T, D)
    want = oracle(x.reshape(-1, D), gate.reshape(-1, D), None, [(b * T, (b + 1) * T) for b in range(B)])
    h, state = gated_scan(x[:, :150], gate[:, :150], return_state=True)
    assert torch.equal(state.to(dtype), h[:, -1])
    rows = [h]
    with torch.no_grad():
        for t in range(150, T):
            rows.append(gated_scan_step_(state, x[:, t], gate[:, t])[:, None])
    near(torch.cat(rows, 1), want["h"], "h")
    near(state, want["final"], "final")
    # rows of a larger state, the version counter
    big = torch.zeros(8, D + 4, device=DEV)
    version = big._version
    out = gated_scan_step_(big[2:7, 1:D + 1], x[:, 0], gate[:, 0])
    near(out, [want["h"][0].view(B, T, D)[:, 0], want["h"][1].view(B, T, D)[:, 0]], "first")
    assert big._version > version and float(big[:2].abs().sum() + big[7:].abs().sum() + big[:, 0].abs().sum() + big[:, D + 1:].abs().sum()) == 0.0
    assert gated_scan_step_(big[:0, :D], x[:0, 0], gate[:0, 0]).shape == (0, D)


@gpu
@pytest.mark.parametrize("T,D", [(20000, 72), (100, 72)])
def test_repeats_streams_and_graphs(native, T, D):
    x, gate, dh = inputs(T, D, BF, seed=33)
    leaves = [t.view(1, T, D).detach().requires_grad_(True) for t in (x, gate)]
    up = dh.view(1, T, D)

    def run():
        h, final = gated_scan(*leaves, return_state=True)
        return [h.detach(), final.detach(), *torch.autograd.grad(h, leaves, up)]
    want = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):                                   # calls at once
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, run()))
    for graph, held in graphs * 2:
        for v in held:
            v.fill_(float("nan"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    ops.check_status()


@gpu
def test_offsets_are_reported_into_the_buffer_of_the_call(native):
    from streamep_b200.models.moe_layer import make_buffer
    buf = make_buffer(None, 64, 64, 2, 4)
    x, gate, dh = inputs(300, 16, BF, seed=1)
    good = torch.tensor([0, 100, 300], device=DEV)
    assert torch.equal(gated_scan(x, gate, offsets=good, buffer=buf), gated_scan(x, gate, offsets=good))
    buf.check_status()
    gated_scan(x, gate, offsets=torch.tensor([0, 301], device=DEV), buffer=buf)
    ops.check_status()
    with pytest.raises(StreamEPError, match="offsets"):
        buf.check_status()
    buf.check_status()


@gpu
def test_bad_offsets_are_reported(native):
    x, gate, dh = inputs(300, 16, BF, seed=1)
    for at in ([0, 200, 100, 300], [0, 301], [-1, 5], [5, 2], [0, 2 ** 31 - 1]):
        gated_scan(x, gate, offsets=torch.tensor(at, dtype=torch.int32, device=DEV), return_state=True)
        with pytest.raises(StreamEPError, match="offsets"):
            ops.check_status()
        ops.check_status()
    gated_scan(x, gate, offsets=torch.tensor([0, 2 ** 40], device=DEV), return_state=True)
    with pytest.raises(StreamEPError, match="offsets"):
        ops.check_status()


@gpu
def test_refusals(native):
    x, gate = torch.randn(2, 5, 16, device=DEV), torch.randn(2, 5, 16, device=DEV)
    state = torch.zeros(2, 16, device=DEV)
    two = torch.tensor([0, 3, 5], device=DEV)
    for f in (lambda: gated_scan(x[0], gate[0]), lambda: gated_scan(x, gate, offsets=two), lambda: gated_scan(x, gate[:1]), lambda: gated_scan(x, gate.to(BF)),
              lambda: gated_scan(x.half(), gate.half()), lambda: gated_scan(x, gate, initial_state=state[:1]), lambda: gated_scan(x, gate, initial_state=state.to(BF)),
              lambda: gated_scan(x[0], gate[0], offsets=two.float()), lambda: gated_scan(x[0], gate[0], offsets=two.cpu()), lambda: gated_scan(x[0], gate[0], offsets=two[:0]),
              lambda: gated_scan(x[..., :0], gate[..., :0]), lambda: gated_scan(x, gate.cpu()),
              lambda: gated_scan_step_(state, x[:, 0], gate[:, 0].to(BF)), lambda: gated_scan_step_(state.to(BF), x[:, 0], gate[:, 0]),
              lambda: gated_scan_step_(state[:1].expand(2, 16), x[:, 0], gate[:, 0]), lambda: gated_scan_step_(torch.zeros(16, 2, device=DEV).t(), x[:, 0], gate[:, 0]),
              lambda: gated_scan_step_(state, x, gate), lambda: gated_scan_step_(state, state, gate[:, 0]), lambda: gated_scan_step_(state, x[:, 0], state)):
        with pytest.raises(ValueError):
            f()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        gated_scan_step_(state, leaf[:, 0], gate[:, 0])
    h = gated_scan(leaf, gate)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(h.sum(), leaf, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            gated_scan(torch.autograd.forward_ad.make_dual(x, x), gate)
    h = gated_scan(leaf, gate)
    with torch.no_grad():
        h.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(h.sum(), leaf)


def test_refused_without_a_gpu():
    x = torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan_step_(x[0], x[0], x[0])
