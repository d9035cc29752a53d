"""linear_cross_entropy's backward over many pieces of the vocabulary, which take turns in two buffers of dz: small calls with a limit of
their own on a piece."""
import pytest
import torch

from loss_bounds import Gradients
from streamep_b200 import _ext
from streamep_b200.ops import grouped_gemm as gg

DEV = "cuda"
SMS = 148
# tokens, hidden, vocabulary, 256-column tiles of a piece: tokens as rows, as columns, and as columns with dz in two parts; last pieces that are
# full, of one column, and of a few; more and fewer tiles of dx than splits
SIZES = [(700, 136, 1500, 1), (700, 136, 1537, 2), (1000, 264, 3333, 3), (2049, 72, 1281, 1), (260, 520, 6000, 8),
         (300, 136, 1500, 1), (100, 264, 3333, 3), (576, 72, 1537, 2), (160, 520, 9000, 12),
         (40, 136, 1500, 1), (1, 72, 1537, 2), (64, 264, 3333, 3), (33, 520, 9000, 12), (16, 1032, 20000, 26)]


def limit(T, tiles):
    return T * 2 * (2 if T <= 64 else 1) * 256 * tiles


@pytest.mark.parametrize("T,H,V,tiles", SIZES)
def test_sizes_have_pieces_that_take_turns(T, H, V, tiles):
    """On the CPU: so that another limit, or rule, cannot empty the test below."""
    for want_dx, want_dw in ((True, True), (True, False), (False, True)):
        (pieces, piece, _, _, buffers, _, split2, _), *_ = _ext.load().linear_loss_schedule(T, H, V, SMS, want_dx, want_dw, limit(T, tiles))
        assert 3 <= pieces <= 6 and pieces > buffers == 2 and piece % 256 == 0 and split2 == (T <= 64)


def run(x, w, y, up, piece_bytes, want_dx=True, want_dw=True, reduction=0):
    x, w = x.detach().requires_grad_(want_dx), w.detach().requires_grad_(want_dw)
    loss = gg.default_runtime().linear_loss(x, w, y, -100, reduction, piece_bytes)
    wanted = [t for t, k in ((x, want_dx), (w, want_dw)) if k]
    got = list(torch.autograd.grad(loss, wanted, up))
    torch.cuda.synchronize()
    assert gg.default_runtime().poll_status(True) == ""
    return loss.detach(), got.pop(0) if want_dx else None, got[0] if want_dw else None


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,tiles", SIZES)
def test_many_pieces(native, T, H, V, tiles):
    g = torch.Generator(device=DEV).manual_seed(T + V)
    w = (torch.randn(V, H, generator=g, device=DEV) * 0.1).bfloat16()
    x = torch.randn(T, H, generator=g, device=DEV).bfloat16()
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    y[-1] = V - 1
    if T > 1:
        y[T // 2] = -100
    up = torch.randn(T, generator=g, device=DEV)
    small = limit(T, tiles)
    want = Gradients(x, w, y, up)
    for want_dx, want_dw in ((True, True), (True, False), (False, True)):
        loss, gx, gw = run(x, w, y, up, small, want_dx, want_dw)
        want.check(gx, gw)
        for _ in range(5):
            again = run(x, w, y, up, small, want_dx, want_dw)
            assert all(a is b is None or torch.equal(a, b) for a, b in zip(again, (loss, gx, gw)))
    mean = Gradients(x, w, y, torch.full((T,), 0.5, device=DEV) / (y != -100).sum())
    mean.check(*run(x, w, y, torch.tensor(0.5, device=DEV), small, reduction=1)[1:])
    with pytest.raises(ValueError):
        gg.default_runtime().linear_loss(x, w, y, -100, 0, -1)
