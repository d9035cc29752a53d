"""adamw_step_ whose step is a number on the device, and ExpertAdamW's count of the updates it made.

Tolerance of an update in fp32: m, v and the two corrections are a handful of roundings each (2^-24), root, quotient and the last sum as many:
16 roundings, 1e-6 of the sum of the magnitudes, taken as 2e-6."""
import math

import pytest
import torch

from streamep_b200.ops import adamw_step_, grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tensors(n, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    p, g_, m, v = (torch.randn(n, generator=g, device=DEV) for _ in range(4))
    return p, g_, m * 0.1, (v * 0.1).square()


def oracle(p, g, m, v, step, lr, betas, eps, decay):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    b1, b2 = betas
    c1, c2 = -math.expm1(step * math.log(b1)) if b1 else 1.0, -math.expm1(step * math.log(b2)) if b2 else 1.0
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    below = (v2 / c2).sqrt() + eps
    size = p.abs() + lr * (b1 * m.abs() + (1 - b1) * g.abs()) / c1 / below
    return p * (1 - lr * decay) - lr * m2 / c1 / below, size


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.9999), (0.0, 0.999), (0.99, 0.0)])
@pytest.mark.parametrize("step", [1, 2, 37, 100_000, 5_000_000_000])
def test_step_on_the_device(native, step, betas):
    o = dict(lr=0.01, betas=betas, eps=1e-8, weight_decay=0.1)
    for sizes in ([1], [5, 0, 4099, 30_001]):
        lists = [list(x) for x in zip(*(tensors(n, i) for i, n in enumerate(sizes)))]
        want = [oracle(*x, step, 0.01, betas, 1e-8, 0.1) for x in zip(*lists)]
        other = [[t.clone() for t in l] for l in lists]
        count = torch.tensor(step, device=DEV)
        adamw_step_(*lists, step=count, **o)
        adamw_step_(*other, step=step, **o)
        assert int(count) == step
        for got, plain, (w, size) in zip(lists[0], other[0], want):
            assert ((got.double() - w).abs() <= 2e-6 * size).all()
            assert ((plain.double() - w).abs() <= 2e-6 * size).all()
        for a, b in zip(lists[2] + lists[3], other[2] + other[3]):
            assert torch.equal(a, b)


def test_many_tensors_and_masters(native):
    """Two launches, chunks in turn: every block has the step."""
    n, sizes = 700, [20_011 + i for i in range(700)]
    ps, gs, ms, vs = [list(x) for x in zip(*(tensors(k, i) for i, k in enumerate(sizes)))]
    masters = [p.clone() for p in ps]
    ps, gs = [p.bfloat16() for p in ps], [g.bfloat16() for g in gs]
    want = [oracle(w, g, m, v, 3, 0.01, (0.9, 0.95), 1e-8, 0.0) for w, g, m, v in zip(masters, gs, ms, vs)]
    adamw_step_(ps, gs, ms, vs, masters=masters, step=torch.tensor([3], device=DEV), lr=0.01, betas=(0.9, 0.95))
    for i in range(n):
        assert ((masters[i].double() - want[i][0]).abs() <= 2e-6 * want[i][1]).all()
        assert torch.equal(ps[i], masters[i].bfloat16())


def test_replayed_graph_counts(native):
    """A captured update whose count is raised in the graph makes update 1, 2, 3 when it is replayed."""
    p, g, m, v = tensors(5000, 7)
    m.zero_()
    v.zero_()
    q, qm, qv = p.clone(), m.clone(), v.clone()
    count = torch.zeros((), dtype=torch.int64, device=DEV)
    norm = grad_norm([g])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count += norm < math.inf
        adamw_step_([p], [g], [m], [v], step=count, lr=0.01, norm=norm, max_norm=1.0, skip_nonfinite=True)
    for step in (1, 2, 3):
        graph.replay()
        adamw_step_([q], [g], [qm], [qv], step=step, lr=0.01, norm=norm, max_norm=1.0)
        torch.cuda.synchronize()
        assert int(count) == step
        torch.testing.assert_close(p, q, rtol=2e-6, atol=2e-6 * 0.02)
        assert torch.equal(m, qm) and torch.equal(v, qv)
    norm.fill_(float("nan"))
    before = p.clone()
    graph.replay()
    assert torch.equal(p, before) and int(count) == 3


def test_refusals(native):
    p, g, m, v = tensors(100, 0)
    for step in (0, -1, torch.tensor(1), torch.tensor(1.0, device=DEV), torch.tensor(1, dtype=torch.int32, device=DEV), torch.tensor([1, 2], device=DEV)):
        with pytest.raises(ValueError):
            adamw_step_([p], [g], [m], [v], step=step, lr=0.1)


def test_skipped_updates_are_not_counted(native):
    """A first step that is left out for its infinite norm, and another later: the updates between are those of an optimizer that never saw them."""
    from streamep_b200.models import ExpertAdamW
    gen = torch.Generator(device=DEV).manual_seed(0)
    params = [torch.randn(n, generator=gen, device=DEV).bfloat16().requires_grad_(True) for n in (1000, 37)]
    opt = ExpertAdamW(params[:1], params[1:], lr=1e-2)
    twin = [m.clone().requires_grad_(True) for m in opt.masters]
    ref = torch.optim.AdamW(twin, lr=opt.lr, betas=opt.betas, eps=opt.eps, weight_decay=opt.weight_decay)
    for i in range(5):
        grads = [torch.randn(p.shape, generator=gen, device=DEV).bfloat16() for p in params]
        for p, g in zip(params, grads):
            p.grad = g
        if i in (0, 3):
            grads[1][5] = float("nan") if i else float("inf")
            before = [t.clone() for t in opt.masters + opt.exp_avgs + opt.exp_avg_sqs]
            opt.step()
            assert all(torch.equal(a, b) for a, b in zip(before, opt.masters + opt.exp_avgs + opt.exp_avg_sqs))
            continue
        for t, g in zip(twin, grads):
            t.grad = g.float()
        torch.nn.utils.clip_grad_norm_(twin, opt.max_norm)
        ref.step()
        opt.step()
        for got, want in zip(opt.masters, twin):
            torch.testing.assert_close(got, want.detach(), rtol=1e-5, atol=2e-5 * opt.lr)
    other = ExpertAdamW([p.detach().clone().requires_grad_(True) for p in params[:1]], [p.detach().clone().requires_grad_(True) for p in params[1:]], lr=1e-2)
    other.load_state_dict(opt.state_dict())
    for a, b in zip(other.params, params):
        a.grad = b.grad = torch.ones_like(b)
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(opt.masters, other.masters))
