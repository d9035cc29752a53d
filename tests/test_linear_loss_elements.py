"""linear_cross_entropy's gradients element by element: what no target's row or column covers up, and sums that cancel."""
import pytest
import torch

from loss_bounds import Gradients
from streamep_b200.ops import check_status, linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(T, H, V, seed, std=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return ((torch.randn(T, H, generator=g, device=DEV)).bfloat16(), (torch.randn(V, H, generator=g, device=DEV) * std).bfloat16(),
            torch.randint(0, V, (T,), generator=g, device=DEV), torch.randn(T, generator=g, device=DEV))


def run(x, w, y, up, reduction="none"):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    got = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction=reduction), (x, w), up)
    check_status()
    return got


# one token to a tile more than three; vocabularies that a few tokens reach nearly nothing of, and such as cancel (few columns, weights of both signs)
SIZES = [(1, 64, 2000), (30, 72, 30001), (64, 64, 100_003), (65, 320, 777), (200, 136, 40_000), (300, 72, 30001), (576, 136, 2049), (577, 72, 20_000),
         (1000, 136, 33000), (640, 192, 70000), (1024, 64, 131073), (2049, 264, 2500),
         (293, 8, 6), (727, 8, 9), (128, 40, 13), (40, 8, 5), (300, 24, 2), (1000, 16, 4)]


@pytest.mark.parametrize("T,H,V", SIZES)
def test_every_element(native, T, H, V):
    x, w, y, up = make(T, H, V, T + V)
    y[T // 3] = -100 if T > 1 else 0
    want = Gradients(x, w, y, up)
    gx, gw = run(x, w, y, up)
    want.check(gx, gw)
    # rows of dW that are no token's target, and those that are, on their own
    target = torch.zeros(V, dtype=torch.bool, device=DEV)
    target[y[y >= 0]] = True
    for rows in (target, ~target):
        if rows.any():
            want.check_norm(gw[rows], want.dw[rows], want.dw_rss[rows], want.dw_worst[rows])
    one = torch.tensor(-0.3, device=DEV)
    mean = Gradients(x, w, y, (one / (y >= 0).sum()).expand(T))
    mean.check(*run(x, w, y, one, "mean"))


@pytest.mark.parametrize("T,H,V", [s for s in SIZES if s[2] >= 500])
def test_dx_without_the_targets_rows(native, T, H, V):
    """The targets' rows of the projection are zeros: dx is the sum over all other columns, which those rows else cover up."""
    x, w, y, up = make(T, H, V, T * V % 1000)
    rows = torch.tensor([0, V // 2, V - 1], device=DEV)
    w[rows] = 0
    y = rows[y % 3]
    Gradients(x, w, y, up).check(*run(x, w, y, up))
