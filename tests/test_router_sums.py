"""balanced_router's sums over many tokens."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.ops import balanced_router

gpu = pytest.mark.gpu
DEV = "cuda"


@gpu
@pytest.mark.parametrize("H", [18944, 37888])
def test_dw_of_many_tokens_is_not_too_small(native, H):
    """All tokens alike, so that every term of an element of dW has one sign, and what an accumulator cuts off adds up.  A part has 4096 tokens at most:
    256 steps of 16, twice for the two numbers of dz.  A step adds 16 products and what was there, aligned to the largest of them; in 24 bits each loses up to
    2^-23 of that one, 17 2^-23 of the sum so far, 17 2^-24 of the final one on average.  Parts are joined by up to 40 sums; dz itself is
    off by 2^-16 (two bf16 numbers) and 2^-20 (exponentials, products).  The result is that sum rounded, and rounding keeps order: it lies between
    the rounded ends of the sum's range.  (A result's own rounding is up to 2^-8 of it, and hides a smaller error in all but the elements next to a border.)"""
    T, E = 1 << 17, 2
    slack = (512 * 17 + 40) * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -20
    g = torch.Generator(device=DEV).manual_seed(1)
    row = (0.5 + torch.rand(H, generator=g, device=DEV)).to(torch.bfloat16)
    x = row.expand(T, H).contiguous()
    w = torch.zeros(E, H, device=DEV, dtype=torch.bfloat16)
    w[0, 0] = 0.3
    w.requires_grad_(True)
    route = balanced_router(x, w, 1, renormalize=False)
    assert bool((route.topk_idx == 0).all())
    p = torch.softmax(row.double() @ w.detach().double().t(), 0)
    for i in range(24):
        up = torch.full((T, 1), (1 + 0.04 * i) / T, device=DEV)
        dw, = torch.autograd.grad(route.topk_weights, w, up, retain_graph=True)
        d = p[0] * (p.new_tensor([1.0, 0.0]) - p) * up[0, 0].double() * T
        want = (d[:, None] * row.double()).abs()
        got = dw * torch.tensor([[1], [-1]], device=DEV)
        least, most = ((want * (1 + sign * slack)).to(torch.bfloat16) for sign in (-1, 1))
        assert bool((got >= least).all()) and bool((got <= most).all()), (i, int((got < least).sum()), int((got > most).sum()))
    ops.check_status()


@gpu
def test_losses_of_many_tokens(native):
    """All tokens alike, so that the sums of all blocks are, and a plain sum of them would round to one side for long stretches.  In units of 2^-24: a
    probability is off by 4 (exponential), 15 (its sum: 10 of a lane, 5 steps over the warp) and 3; a block's sum by 4 tokens of a warp and 16 warps; the sum of
    all blocks keeps what it loses, and 3 rows and 5 steps join it; the load and products 6.  The squared logsumexp: twice 20, and its sums the same way."""
    T, H, E = 1 << 21, 8, 300
    slack = 64 * 2.0 ** -24
    for i in range(6):
        x = torch.zeros(T, H, device=DEV, dtype=torch.bfloat16)
        w = torch.zeros(E, H, device=DEV, dtype=torch.bfloat16)
        x[:, 0], w[0, 0] = 1.0, 5.0 + i * 0.375
        route = balanced_router(x, w, 1)
        z = x[0].double() @ w.double().t()
        assert int(route.expert_counts[0]) == T
        assert abs(float(route.balance_loss) / float(E * torch.softmax(z, 0)[0]) - 1) <= slack
        assert abs(float(route.z_loss) / float(torch.logsumexp(z, 0) ** 2) - 1) <= slack
    ops.check_status()
