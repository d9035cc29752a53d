"""balanced_router against 64-bit arithmetic: expert counts around warps and tiles, token counts around blocks, masks (none counts, one
counts), weights with and without their second softmax, each subset of gradients, streams, captured graphs, refusals.

Inputs: small whole numbers times powers of two, with logits on a grid of 1/64, so that every logit is exact in 32 bits and its order no matter of
rounding; ties are frequent and go to the lowest expert.

Tolerances.  A probability's exponential is off by 2^-22 of itself and, through its argument, by 2^-24 of 2 |z|max; its sum and
quotient add E / 32 + 8 roundings: P = (E / 32 + 14 + 2 |z|max) 2^-24 of itself.  Means over tokens add T / 16 + 160 roundings.  dz, a handful of
products of such values, is off by 4 P of D, the sum of its terms' magnitudes; the products round dz to bf16 at most (2^-8 of D), and add in fp32
(2^-22 for each of their 64-element steps).  Results in bf16 are rounded once."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.ops import balanced_router, router_topk

gpu = pytest.mark.gpu
DEV = "cuda"
BF, F64 = torch.bfloat16, torch.float64
ULP = 2.0 ** -24


def inputs(T, H, E, seed=0):
    """x has a few non-zero entries of 1/8 a row, w_gate entries of 1/8: logits are multiples of 1/64 up to a few units."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-24, 25, (T, H), generator=g, device=DEV) / 8.0
    x = x * (torch.rand(T, H, generator=g, device=DEV) < min(1.0, 12.0 / H))
    w = torch.randint(-8, 9, (E, H), generator=g, device=DEV) / 8.0
    return x.to(BF), w.to(BF)


def near(got, want, slack, what):
    half = torch.finfo(got.dtype).eps / 2
    over = (got.double() - want).abs() - (slack + half * want.abs())
    assert got.shape == want.shape and bool((over <= 0).all()), f"{what}: {float(over.max()):.3e} above the bound"


def oracle(x, w, K, R, renormalize, mask, ups=None):
    T, E = x.shape[0], w.shape[0]
    z = x.double() @ w.double().t()
    p = torch.softmax(z, 1)
    # probabilities of equal logits are equal, and so are those that round to the same number: the order of the logits, lowest first
    idx = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :K]
    chosen = p.gather(1, idx)
    wts = chosen / chosen.sum(1, keepdim=True) if renormalize else chosen
    in_rank = torch.zeros(T, R, dtype=torch.bool, device=DEV)
    in_rank[torch.arange(T, device=DEV)[:, None], idx // (E // R)] = True
    m = mask if mask is not None else torch.ones(T, dtype=torch.bool, device=DEV)
    n = int(m.sum())
    share = 1.0 / n if n else 0.0
    counts = torch.bincount(idx[m].reshape(-1), minlength=E)
    load = counts.double() * E / K * share
    lse = torch.logsumexp(z, 1)
    balance = (load * p[m].sum(0) * share).sum()
    zl = lse[m].square().sum() * share
    out = dict(z=z, p=p, idx=idx, weights=wts, in_rank=in_rank, counts=counts, balance=balance, zl=zl)
    if ups is None:
        return out
    up, db, dzl = ups
    dz, D = torch.zeros_like(p), torch.zeros_like(p)
    if up is not None:
        up = up.double()
        mean, size = (wts * up).sum(1, keepdim=True), (wts * up.abs()).sum(1, keepdim=True)
        if renormalize:
            dz.scatter_add_(1, idx, wts * (up - mean))
            D.scatter_add_(1, idx, wts * (up.abs() + size))
        else:
            dz.scatter_add_(1, idx, chosen * up)
            D.scatter_add_(1, idx, chosen * up.abs())
            dz -= p * mean
            D += p * size
    on = m.double()[:, None] * share
    if db is not None:
        inner = (p * load).sum(1, keepdim=True)
        dz += float(db) * on * p * (load - inner)
        D += abs(float(db)) * on * p * (load + inner)
    if dzl is not None:
        dz += 2 * float(dzl) * on * lse[:, None] * p
        D += 2 * abs(float(dzl)) * on * lse.abs()[:, None] * p
    out.update(dz=dz, D=D, dx=dz @ w.double(), dw=dz.t() @ x.double())
    return out


def check(T, H, E, K, R=1, renormalize=True, masked=None, which=7, seed=0):
    x, w = inputs(T, H, E, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    mask = None if masked is None else torch.rand(T, generator=g, device=DEV) >= masked
    up = torch.randn(T, K, generator=g, device=DEV)
    db, dzl = torch.tensor(0.7 * T, device=DEV), torch.tensor(-0.3 * T, device=DEV)
    ups = [u if which >> i & 1 else None for i, u in enumerate((up, db, dzl))]
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = balanced_router(xl, wl, K, R, renormalize, mask=mask)
    want = oracle(x, w, K, R, renormalize, mask, ups)
    assert torch.equal(r.topk_idx, want["idx"]) and torch.equal(r.is_token_in_rank, want["in_rank"]) and torch.equal(r.expert_counts, want["counts"])
    assert r.expert_counts.dtype == torch.int64 and r.balance_loss.shape == () and r.z_loss.shape == ()
    P = (E / 32 + 14 + 2 * float(want["z"].abs().max() if T else 0.0)) * ULP
    near(r.topk_weights.detach(), want["weights"], (2 * P + K * ULP) * want["weights"], "weights")
    A = P + (T / 16 + 160) * ULP
    near(r.balance_loss.detach(), want["balance"], (A + E * ULP) * want["balance"], "balance")
    near(r.z_loss.detach(), want["zl"], 2 * A * (want["zl"] + want["zl"].sqrt()), "z")
    outs = [o for i, o in enumerate((r.topk_weights, r.balance_loss, r.z_loss)) if which >> i & 1]
    dx, dw = torch.autograd.grad(outs, [xl, wl], [u for u in ups if u is not None])
    rel = 2.0 ** -8 + 4 * P + A
    near(dx, want["dx"], (rel + E / 64 * 2.0 ** -22) * (want["D"] @ w.double().abs()), "dx")
    near(dw, want["dw"], (rel + (T / 64 + 8) * 2.0 ** -22) * (want["D"].t() @ x.double().abs()), "dw")
    assert dx.dtype == BF and dw.dtype == BF
    ops.check_status()
    return r, dx, dw


@gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,K,R", [(1, 1, 1), (2, 2, 2), (8, 2, 8), (8, 6, 1), (31, 4, 1), (32, 1, 4), (60, 3, 4), (64, 6, 8), (100, 8, 2), (128, 32, 1), (129, 5, 1),
                                   (256, 8, 8), (320, 7, 5), (512, 8, 32)])
def test_experts(native, E, K, R, renormalize):
    check(200, 256, E, K, R, renormalize, seed=E)
    check(131, 136, E, K, R, renormalize, masked=0.4, seed=E + 1)


@gpu
@pytest.mark.parametrize("T", [0, 1, 2, 15, 16, 17, 63, 65, 127, 128, 129, 1000, 4097])
@pytest.mark.parametrize("E,K", [(64, 6), (160, 4)])
def test_tokens(native, T, E, K):
    check(T, 512, E, K, seed=T)
    check(T, 72, E, K, masked=0.5, renormalize=False, seed=T)


@gpu
@pytest.mark.parametrize("H", [8, 16, 56, 64, 72, 120, 128, 200, 1000, 2048, 4104])
def test_hidden(native, H):
    check(150, H, 64, 4, seed=H)
    check(300, H, 24, 2, masked=0.2, seed=H)


@gpu
@pytest.mark.parametrize("T,H,E", [(3329, 7176, 100), (3457, 7160, 128), (3400, 4104, 200), (1537, 4128, 512), (2049, 8000, 257), (9473, 1032, 256),
                                   (9729, 1304, 130), (19000, 1096, 160), (9500, 1024, 200), (2400, 7176, 200), (4100, 4360, 512), (8200, 2056, 129)])
def test_many_weights(native, T, H, E):
    """Products of which two blocks share the work: an odd count of blocks, tokens and columns that end inside."""
    check(T, H, E, 4, masked=0.1, seed=E)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(1, 8))
def test_subsets_of_upstream_gradients(native, which):
    for renormalize in (True, False):
        check(300, 128, 40, 3, renormalize=renormalize, masked=0.3, which=which, seed=which)


@gpu
def test_subsets_of_inputs(native):
    x, w = inputs(500, 320, 64, 3)
    g = torch.Generator(device=DEV).manual_seed(1)
    up = torch.randn(500, 4, generator=g, device=DEV)

    def grads(a, b):
        xl, wl = x.clone().requires_grad_(a), w.clone().requires_grad_(b)
        r = balanced_router(xl, wl, 4)
        return torch.autograd.grad([r.topk_weights, r.balance_loss], [v for v, on in ((xl, a), (wl, b)) if on], [up, torch.ones((), device=DEV)])
    both = grads(True, True)
    assert torch.equal(grads(True, False)[0], both[0]) and torch.equal(grads(False, True)[0], both[1])


@gpu
def test_masks(native):
    x, w = inputs(700, 128, 64, 5)
    none = balanced_router(x, w, 4, mask=torch.zeros(700, dtype=torch.bool, device=DEV))
    assert float(none.balance_loss) == 0.0 and float(none.z_loss) == 0.0 and int(none.expert_counts.sum()) == 0
    check(700, 128, 64, 4, masked=1.1)                   # nothing counts: only the weights' gradients are left
    check(700, 128, 64, 4, masked=1.1, which=6)
    full, plain = balanced_router(x, w, 4, mask=torch.ones(700, dtype=torch.bool, device=DEV)), balanced_router(x, w, 4)
    assert all(torch.equal(a, b) for a, b in zip(full, plain))
    idx, weights, in_rank = router_topk(x, w, 4)
    assert torch.equal(idx, plain.topk_idx) and torch.equal(in_rank, plain.is_token_in_rank)
    torch.testing.assert_close(weights, plain.topk_weights, rtol=1e-5, atol=0.0)           # (its exponentials are coarser: 2^-20 here)
    # padding holds anything at all
    mask = torch.ones(700, dtype=torch.bool, device=DEV)
    mask[600:] = False
    bad = x.clone()
    bad[650:] = float("nan")
    bad[640:650] = float("inf")
    a, b = balanced_router(x, w, 4, mask=mask), balanced_router(bad, w, 4, mask=mask)
    assert torch.equal(a.balance_loss, b.balance_loss) and torch.equal(a.z_loss, b.z_loss) and torch.equal(a.expert_counts, b.expert_counts)
    assert torch.equal(a.topk_weights[:600], b.topk_weights[:600])
    every = mask.repeat_interleave(2)[::2]               # a mask with gaps in memory
    assert not every.is_contiguous() and torch.equal(balanced_router(x, w, 4, mask=every).balance_loss, a.balance_loss)


@gpu
def test_places(native):
    x, w = inputs(90, 64, 32, 8)
    up = torch.randn(90, 2, device=DEV)

    def run(x, w):
        xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        r = balanced_router(xl, wl, 2)
        return [v.detach() for v in r] + list(torch.autograd.grad([r.topk_weights, r.z_loss], [xl, wl], [up, torch.ones((), device=DEV)]))
    want = run(x, w)
    odd = lambda t: torch.cat([torch.zeros(1, device=DEV, dtype=BF), t.reshape(-1)])[1:].view(t.shape)
    wide = lambda t: torch.cat([t, t], 1)[:, :t.shape[1]]
    turned = lambda t: t.t().contiguous().t()
    for f in (odd, wide, turned):
        assert all(torch.equal(a, b) for a, b in zip(run(f(x), f(w)), want))


@gpu
def test_against_differences(native):
    """Logits are products in 32 bits of bf16 numbers, so steps along x and w_gate are steps of bf16: whole powers of two."""
    T, H, E, K = 40, 64, 16, 3
    g = torch.Generator(device=DEV).manual_seed(2)
    x = (torch.randint(-16, 17, (T, H), generator=g, device=DEV) / 16.0).to(BF)
    w = (torch.randint(-16, 17, (E, H), generator=g, device=DEV) / 32.0).to(BF)
    up, db, dzl = torch.randn(T, K, generator=g, device=DEV), 20.0, 5.0
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = balanced_router(xl, wl, K)
    grads = torch.autograd.grad([r.topk_weights, r.balance_loss, r.z_loss], [xl, wl], [up, torch.tensor(db, device=DEV), torch.tensor(dzl, device=DEV)])
    idx, counts = r.topk_idx, r.expert_counts

    def value(a, b):                                     # with the choice held, as the gradient has it
        z = a.double() @ b.double().t()
        p = torch.softmax(z, 1)
        c = p.gather(1, idx)
        return float((c / c.sum(1, keepdim=True) * up.double()).sum() + db * E * (counts.double() / (K * T) * p.mean(0)).sum()
                     + dzl * torch.logsumexp(z, 1).square().mean())
    for i, (t, grad) in enumerate(((x, grads[0]), (w, grads[1]))):
        v = torch.randint(-1, 2, t.shape, generator=g, device=DEV).double()
        h = 2.0 ** -10
        at = lambda f: value(*(q.double() + (f * h * v if k == i else 0.0) for k, q in enumerate((x, w))))
        exact, twice = (at(1) - at(-1)) / (2 * h), (at(2) - at(-2)) / (4 * h)
        slope = float((grad.double() * v).sum())
        # the gradient's own bound, element by element, and the differences' error of second order
        want = oracle(x, w, K, 1, True, None, (up, db, dzl))
        D = want["D"] @ w.double().abs() if i == 0 else want["D"].t() @ x.double().abs()
        bound = float(((2.0 ** -8 + 2.0 ** -16) * (D + grad.double().abs()) * v.abs()).sum())
        assert abs(slope - exact) <= bound + abs(exact - twice)


@gpu
def test_gradients_of_losses_where_padding_holds_anything(native):
    """At sizes whose products are shared by blocks, and below."""
    for T, H, E in ((700, 128, 64), (9601, 2056, 200)):
        x, w = inputs(T, H, E, 5)
        mask = torch.ones(T, dtype=torch.bool, device=DEV)
        mask[T // 2 + 50:T // 2 + 150] = False
        bad = x.clone()
        bad[T // 2 + 50:T // 2 + 100] = float("nan")
        bad[T // 2 + 100:T // 2 + 150] = float("inf")
        grads = []
        for rows in (x, bad):
            xl, wl = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
            r = balanced_router(xl, wl, 4, mask=mask)
            grads.append(torch.autograd.grad([r.balance_loss, r.z_loss], [xl, wl], [torch.tensor(3.0 * T, device=DEV)] * 2))
        # (a row of x that is infinite or NaN times a gradient of zero is NaN, for the experts of dW that it meets: only dx is the same)
        assert torch.equal(grads[0][0], grads[1][0]) and bool((grads[0][0][~mask] == 0).all())


@gpu
@pytest.mark.parametrize("T,H,E", [(3000, 512, 64), (9601, 2056, 200)])
def test_repeats_streams_and_graphs(native, T, H, E):
    x, w = inputs(T, H, E, 9)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    up = torch.randn(T, 6, device=DEV)

    def run():
        r = balanced_router(xl, wl, 6, 8)
        return [v.detach() for v in r] + list(torch.autograd.grad([r.topk_weights, r.balance_loss, r.z_loss], [xl, wl],
                                                                  [up, torch.ones((), device=DEV), torch.ones((), device=DEV)]))
    want = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
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
            v.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    ops.check_status()


@gpu
def test_refusals(native):
    x, w = inputs(10, 64, 16)
    for f in (lambda: balanced_router(x.float(), w, 2), lambda: balanced_router(x, w.float(), 2), lambda: balanced_router(x[:, :32], w, 2),
              lambda: balanced_router(x[None], w, 2), lambda: balanced_router(x, w, 17), lambda: balanced_router(x, w, 0), lambda: balanced_router(x, w, 2, 3),
              lambda: balanced_router(x, w, 2, 0), lambda: balanced_router(x[:, :12], w[:, :12], 2), lambda: balanced_router(x, w[:0], 1),
              lambda: balanced_router(x, w, 2, mask=torch.ones(9, dtype=torch.bool, device=DEV)), lambda: balanced_router(x, w, 2, mask=torch.ones(10, device=DEV)),
              lambda: balanced_router(x, torch.zeros(513, 64, device=DEV, dtype=BF), 2), lambda: balanced_router(x, w.cpu(), 2)):
        with pytest.raises(ValueError):
            f()
    xl = x.clone().requires_grad_(True)
    r = balanced_router(xl, w, 2)
    assert not r.topk_idx.requires_grad and not r.expert_counts.requires_grad and not r.is_token_in_rank.requires_grad and r.topk_weights.requires_grad
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(r.z_loss, xl, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            balanced_router(torch.autograd.forward_ad.make_dual(x, x), w, 2)


def test_refused_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        balanced_router(torch.zeros(4, 8, dtype=BF), torch.zeros(4, 8, dtype=BF), 2)
