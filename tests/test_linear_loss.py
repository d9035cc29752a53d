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
         (448, 512, 1025), (449, 512, 1025), (640, 192, 70000), (1024, 64, 131073), (1025, 72, 2000)]


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
