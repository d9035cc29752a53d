"""ExpertAdamW on the host: what it keeps and what it hands on, with the native calls replaced by their definitions on the CPU."""
import os
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from streamep_b200 import _ext
from streamep_b200.models import ExpertAdamW


class Native:
    """The native calls by their definitions, in 64 bits."""

    @staticmethod
    def list_norm(ts):
        s = sum((t.double().square().sum() for t in ts), torch.zeros((), dtype=torch.float64))
        return s.sqrt().float(), s

    @staticmethod
    def list_adamw(params, grads, exp_avgs, exp_avg_sqs, masters, norm, step, device_step, lr, beta1, beta2, eps, decay, max_norm, skip):
        places = [t.data_ptr() for l in (params, exp_avgs, exp_avg_sqs, masters) for t in l if t.numel()]
        if len(set(places)) != len(places):
            raise ValueError("two tensors that are written in place share memory")
        t = int(device_step) if device_step is not None else step
        f = min(1.0, max_norm / (float(norm) + 1e-6)) if max_norm >= 0 else 1.0
        if skip and not torch.isfinite(norm):
            return
        for p, g, m, v, w in zip(params, grads, exp_avgs, exp_avg_sqs, masters):
            g = g.double() * f
            m.copy_(beta1 * m.double() + (1 - beta1) * g)
            v.copy_(beta2 * v.double() + (1 - beta2) * g * g)
            w.copy_(w.double() * (1 - lr * decay) - lr * (m.double() / (1 - beta1 ** t)) / ((v.double() / (1 - beta2 ** t)).sqrt() + eps))
            p.copy_(w)


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(_ext, "load", lambda: Native)


def torch_twin(opt):
    twin = [m.clone().requires_grad_(True) for m in opt.masters]
    return twin, torch.optim.AdamW(twin, lr=opt.lr, betas=opt.betas, eps=opt.eps, weight_decay=opt.weight_decay)


def follow(opt, twin, ref, grads):
    """One step of both; a gradient of None is none."""
    for p, t, g in zip(opt.params, twin, grads):
        p.grad = None if g is None else g.to(p.dtype)
        t.grad = None if g is None else g.to(p.dtype).to(torch.float32, copy=True)
    if opt.max_norm is not None:
        torch.nn.utils.clip_grad_norm_([t for t in twin if t.grad is not None], opt.max_norm)
    ref.step()
    opt.step()
    for got, want in zip(opt.masters, twin):       # 32-bit arithmetic of the reference: a few 1e-7 of the value, and of a step
        torch.testing.assert_close(got, want.detach(), rtol=1e-6, atol=1e-5 * opt.lr)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masters_are_copies(dtype):
    """Parameters of the masters' own type as well: both are written in a step."""
    params = [torch.randn(50).to(dtype).requires_grad_(True), torch.randn(7).bfloat16().requires_grad_(True)]
    opt = ExpertAdamW(params[:1], params[1:], lr=1e-2)
    assert all(m.dtype == torch.float32 and m.data_ptr() != p.data_ptr() for m, p in zip(opt.masters, params))
    twin, ref = torch_twin(opt)
    for _ in range(3):
        follow(opt, twin, ref, [torch.randn(50), torch.randn(7)])
    for p, m in zip(params, opt.masters):
        assert torch.equal(p.detach(), m.to(p.dtype))


def test_parameters_that_join_late_or_pause():
    """Each parameter's corrections go by its own updates, as the reference optimizer has it."""
    torch.manual_seed(0)
    params = [torch.randn(n).bfloat16().requires_grad_(True) for n in (50, 7, 30)]
    opt = ExpertAdamW(params[:1], params[1:], lr=1e-2)
    twin, ref = torch_twin(opt)
    for mask in ((1, 1, 0), (1, 1, 0), (1, 1, 1), (1, 0, 1), (0, 1, 0), (0, 0, 0), (1, 1, 1)):
        if any(mask):
            follow(opt, twin, ref, [torch.randn(p.shape) if m else None for p, m in zip(params, mask)])
        else:
            opt.zero_grad()
            assert float(opt.step()) == 0.0
    assert opt.state_dict()["steps"].tolist() == [5, 5, 3] and len({id(s) for s in opt.steps}) <= 3
    other = ExpertAdamW([params[0].detach().clone().requires_grad_(True)], [p.detach().clone().requires_grad_(True) for p in params[1:]], lr=1e-2)
    other.load_state_dict(opt.state_dict())
    for a, b in zip(params, other.params):
        a.grad = b.grad = torch.ones_like(b)
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(opt.masters, other.masters))
    other.load_state_dict({**opt.state_dict(), "steps": 4})                         # one number for all
    assert other.state_dict()["steps"].tolist() == [4, 4, 4]


def _rank(rank, world, store, out):
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world)
    _ext.load = lambda: Native
    shared, mine = weights(rank)
    opt = ExpertAdamW(shared, mine, lr=1e-2, max_norm=1.0, group=dist.group.WORLD)
    norms = []
    for step in range(3):
        for p, g in zip(shared + mine, gradients(rank, step)):
            p.grad = None if g is None else g.clone()
        norms.append(float(opt.step()))
    torch.save((norms, opt.masters, opt.state_dict()["steps"]), f"{out}.{rank}")
    dist.destroy_process_group()


def weights(rank):
    g = torch.Generator().manual_seed(1)
    shared = [torch.randn(n, generator=g).requires_grad_(True) for n in (40, 3)]
    g = torch.Generator().manual_seed(10 + rank)
    return shared, [torch.randn(n, generator=g).requires_grad_(True) for n in (20, 11)]


def gradients(rank, step):
    """The second replicated parameter is without one in the middle step, rank 1's last expert in all."""
    g = torch.Generator().manual_seed(100 * step + rank)
    a, b, c, d = (torch.randn(n, generator=g) for n in (40, 3, 20, 11))
    return a, None if step == 1 else b, c, None if rank == 1 else d


def test_step_over_a_group():
    """Two ranks against one process with all experts: replicated gradients are means, the experts' the sum over all tokens divided by the ranks."""
    world = 2
    with tempfile.TemporaryDirectory() as d:
        out = os.path.join(d, "out")
        mp.spawn(_rank, args=(world, os.path.join(d, "store"), out), nprocs=world)
        got = [torch.load(f"{out}.{r}") for r in range(world)]
    shared = weights(0)[0]
    params = shared + weights(0)[1] + weights(1)[1]
    masters = [p.detach().clone().requires_grad_(True) for p in params]
    ref = torch.optim.AdamW(masters, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    for step in range(3):
        a, b = gradients(0, step), gradients(1, step)
        grads = [None if x is None else (x + y) / 2 for x, y in zip(a[:2], b[:2])] + [None if x is None else x / 2 for x in a[2:] + b[2:]]
        for m, g in zip(masters, grads):
            m.grad = g
        norm = float(torch.nn.utils.clip_grad_norm_([m for m in masters if m.grad is not None], 1.0))
        ref.step()
        assert all(abs(norms[step] - norm) <= 1e-5 * norm for norms, _, _ in got)
    for rank, (_, mine, steps) in enumerate(got):
        assert steps.tolist() == [3, 2, 3, 0 if rank == 1 else 3]
        for m, want in zip(mine, masters[:2] + masters[2 + 2 * rank:4 + 2 * rank]):
            torch.testing.assert_close(m, want.detach(), rtol=1e-6, atol=1e-5 * 1e-2)
