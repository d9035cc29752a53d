"""Tensors of more than 2^31 elements: what the last rows get is what they get by themselves."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.ops import balanced_router, gated_scan, gated_scan_step_, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def release():
    yield
    torch.cuda.empty_cache()


def test_normalisation(native):
    rows, H, n = (1 << 18) + 37, 8200, 50
    block = lambda: torch.randn(rows // 8 + 1, H, device=DEV).to(BF).repeat(8, 1)[:rows]
    for H in (8192, 8200):
        x, dy = block(), block()
        assert x.numel() > 1 << 31
        w = torch.randn(H, device=DEV)
        xl = x.requires_grad_(True)
        y = layer_norm(xl, w)
        dx, = torch.autograd.grad(y, xl, dy)
        tail = x.detach()[-n:].clone().requires_grad_(True)
        ty = layer_norm(tail, w)
        assert torch.equal(y.detach()[-n:], ty.detach())
        assert torch.equal(dx[-n:], torch.autograd.grad(ty, tail, dy[-n:])[0])
        del x, dy, xl, y, dx


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("D", [2048, 2049])
def test_recurrence(native, D, packed):
    """The last rows start from a gate that lets nothing through, so that they do not depend on the million in front; they are rounded elsewhere, as
    time is split otherwise: by 2^-8 of a value twice, and 2^-16 for what 32 bits do."""
    rows, n = (1 << 20) + 4099, 70
    block = lambda: torch.randn(rows // 16 + 1, D, device=DEV).to(BF).repeat(16, 1)[:rows]
    x, gate, dh = block(), block(), block()
    gate[-n] = float("-inf")
    assert x.numel() > 1 << 31
    offsets = torch.tensor([0, 5, rows - 1000, rows], device=DEV) if packed else None
    shape = (rows, D) if packed else (1, rows, D)
    leaves = [t.view(shape).requires_grad_(True) for t in (x, gate)]
    h = gated_scan(*leaves, offsets=offsets)
    grads = torch.autograd.grad(h, leaves, dh.view(shape))
    tails = [t.detach()[-n:].clone()[None].requires_grad_(True) for t in (x, gate)]
    th = gated_scan(*tails)
    tg = torch.autograd.grad(th, tails, dh[-n:][None])
    ops.check_status()
    close = lambda a, b: torch.testing.assert_close(a.reshape(rows, D)[-n + 1:].float(), b[0, 1:].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    close(h.detach(), th.detach())
    for a, b in zip(grads, tg):
        close(a, b)
    assert bool(h.detach().isfinite().all()) and bool(grads[0].isfinite().all())


def test_steps(native):
    S, D = (1 << 20) + 11, 2056
    x = torch.randn(S // 16 + 1, D, device=DEV).to(BF).repeat(16, 1)[:S]
    state = torch.zeros(S, D, device=DEV)
    assert x.numel() > 1 << 31
    h = gated_scan_step_(state, x, x)
    small = torch.zeros(9, D, device=DEV)
    assert torch.equal(h[-9:], gated_scan_step_(small, x[-9:], x[-9:])) and torch.equal(state[-9:], small)


def test_routing(native):
    T, H, E = (1 << 20) + 77, 2056, 60
    x = (torch.randint(-8, 9, (T // 16 + 1, H), device=DEV) / 8.0).to(BF).repeat(16, 1)[:T]
    w = (torch.randint(-8, 9, (E, H), device=DEV) / 64.0).to(BF)
    up = torch.randn(T, 4, device=DEV)
    assert x.numel() > 1 << 31
    xl = x.requires_grad_(True)
    r = balanced_router(xl, w, 4)
    dx, = torch.autograd.grad(r.topk_weights, xl, up)
    tail = x.detach()[-77:].clone().requires_grad_(True)
    t = balanced_router(tail, w, 4)
    ops.check_status()
    # (the hidden dimension may be cut otherwise for few tokens: logits are multiples of 2^-9 below 2^8, and exact)
    assert torch.equal(r.topk_idx[-77:], t.topk_idx) and torch.equal(r.topk_weights.detach()[-77:], t.topk_weights.detach())
    assert int(r.expert_counts.sum()) == 4 * T
    got = torch.autograd.grad(t.topk_weights, tail, up[-77:])[0]
    torch.testing.assert_close(dx[-77:].float(), got.float(), rtol=2.0 ** -7, atol=2.0 ** -10)
