"""How many bits balanced_router's products take of the logits' gradient dz: two bf16 numbers up to 128 experts.

A result is rounded to bf16 (2^-8 of it), which would hide an error of dz as large; but rounding keeps order, so a result lies between the rounded ends of the
range of its sum, and the elements next to a border show the rest.  The range, relative to the sum of the terms' magnitudes: 2^-16 (dz), 4 P (its
factors, P = (E / 32 + 14 + 2 |z|max) 2^-24), and for each step of 16 terms that an accumulator takes, of both numbers, 17 2^-23: 17 numbers aligned to the largest
of them and kept to 24 bits at least."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.ops import balanced_router

BF = torch.bfloat16
CASES = [(40, 64, 8, 2), (40, 256, 60, 4), (48, 64, 64, 6), (33, 136, 100, 3), (40, 64, 128, 8)]


def problem(T, H, E, K, device):
    """Weights' gradients without normalisation; logits are exact in 32 bits, and distinct where it matters: ties go to the lowest expert."""
    g = torch.Generator(device="cpu").manual_seed(E)
    x = torch.randint(-24, 25, (T, H), generator=g) / 8.0 * (torch.rand(T, H, generator=g) < min(1.0, 12.0 / H))
    w, up = torch.randint(-8, 9, (E, H), generator=g) / 8.0, torch.randn(T, K, generator=g)
    return x.to(BF).to(device), w.to(BF).to(device), up.to(device)


def ranges(x, w, up, K):
    """{dx, dw}: (least, most) in bf16; and dz."""
    T, E = x.shape[0], w.shape[0]
    a, b, up = x.double(), w.double(), up.double()
    z = a @ b.t()
    p = torch.softmax(z, 1)
    idx = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :K]
    c = p.gather(1, idx)
    dz = torch.zeros_like(p).scatter_add_(1, idx, c * up) - p * (c * up).sum(1, keepdim=True)
    D = torch.zeros_like(p).scatter_add_(1, idx, c * up.abs()) + p * (c * up.abs()).sum(1, keepdim=True)
    P = (E / 32 + 14 + 2 * float(z.abs().max())) * 2.0 ** -24
    rel = lambda n: 2.0 ** -16 + 4 * P + 2 * -(-n // 16) * 17 * 2.0 ** -23
    ends = lambda v, s: ((v - s).to(BF), (v + s).to(BF))
    return {"dx": ends(dz @ b, rel(E) * (D @ b.abs())), "dw": ends(dz.t() @ a, rel(T) * (D.t() @ a.abs()))}, dz


def outside(got, ends):
    return int(((got < ends[0]) | (got > ends[1])).sum())


@pytest.mark.parametrize("T,H,E,K", CASES)
def test_the_range_tells_two_numbers_from_one(T, H, E, K):
    x, w, up = problem(T, H, E, K, "cpu")
    want, dz = ranges(x, w, up, K)
    one = dz.to(BF).double()
    two = one + (dz - one).to(BF).double()
    for kept, right in ((two, True), (one, False)):
        for name, v in (("dx", kept @ w.double()), ("dw", kept.t() @ x.double())):
            assert (outside(v.to(BF), want[name]) == 0) == right, (name, right)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,E,K", CASES)
def test_products_take_two_numbers(native, T, H, E, K):
    x, w, up = problem(T, H, E, K, "cuda")
    want, _ = ranges(x, w, up, K)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    got = torch.autograd.grad(balanced_router(xl, wl, K, renormalize=False).topk_weights, (xl, wl), up)
    ops.check_status()
    for name, v in zip(("dx", "dw"), got):
        assert outside(v, want[name]) == 0, name
