"""Long memories of gated_scan: gates whose state lasts for up to millions of rows.

A state that equals its inputs stays where it is, whatever the gate, since keep + take = 1; a constant gate fades a state by keep^T; and the weights that a
final state gives to its inputs and to the state in front of them add up to 1.  Tolerances, in units of 2^-24 of values of at most one: time is split into
segments of 32 to 128 rows, whose states round once a row, behind the joined runs of those before.  A block joins 4 segments or more, so there are
at most T / 128 of them in a row, and a join rounds four times (b twice, 1 - a twice); `take` itself is off by 8 (exponential 4, sum, reciprocal 2, product)
and, with its exponent rounded once (bf16), by |gate| more: of a weight, and T take of it, at most 0.4 (t e^-t), of a fading state."""
import pytest
import torch

from streamep_b200 import ops
from streamep_b200.ops import gated_scan, gated_scan_step_

gpu = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
T = 300000
SLACK = (128 + 4 * T / 128 + 32) * 2.0 ** -24


def gates(D, dtype):
    return torch.linspace(-4.0, 18.0, D, device=DEV).to(dtype)


def call(x, gate, initial, packed):
    """Two sequences (the rows of both alike), dense or packed behind one another with rows in front that belong to none."""
    if not packed:
        return gated_scan(torch.stack([x, x]), torch.stack([gate, gate]), initial_state=initial, return_state=True)
    rows = lambda t: torch.cat([t[:5], t, t])
    offsets = torch.tensor([5, 5 + T, 5 + 2 * T], device=DEV)
    h, final = gated_scan(rows(x), rows(gate), initial_state=initial, offsets=offsets, return_state=True)
    return h[5:].view(2, T, -1), final


@gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 61), (BF, 64), (BF, 66), (BF, 61)])
def test_a_state_that_equals_its_inputs_stays(native, dtype, D, packed):
    value = (0.5 + torch.arange(D, device=DEV) % 7 / 8.0).to(dtype)
    h, final = call(value.expand(T, D).contiguous(), gates(D, dtype).expand(T, D).contiguous(), value.float().expand(2, D), packed)
    ops.check_status()
    half = torch.finfo(dtype).eps / 2
    assert float((final.double() / value.double() - 1).abs().max()) <= SLACK
    assert float((h.double() / value.double() - 1).abs().max()) <= SLACK + half


@gpu
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 61), (BF, 64), (BF, 66), (BF, 61)])
def test_a_state_fades_at_its_gates_rate(native, dtype, D):
    gate = gates(D, dtype)
    h, final = call(torch.zeros(T, D, device=DEV, dtype=dtype), gate.expand(T, D).contiguous(), torch.ones(2, D, device=DEV), False)
    ops.check_status()
    rate = torch.log1p(-torch.sigmoid(-gate.double()))           # log keep
    want = torch.exp(rate * torch.arange(1, T + 1, device=DEV, dtype=torch.float64)[:, None])
    assert float((final.double() - want[-1]).abs().max()) <= SLACK
    assert float((h.double() - want).abs().max()) <= SLACK + torch.finfo(dtype).eps / 2


@gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 61), (BF, 64), (BF, 66), (BF, 61)])
def test_the_weights_of_a_state_add_up_to_one(native, dtype, D, packed):
    x = torch.zeros(T, D, device=DEV, dtype=dtype, requires_grad=True)
    initial = torch.zeros(2, D, device=DEV, requires_grad=True)
    _, final = call(x, gates(D, dtype).expand(T, D).contiguous(), initial, packed)
    dx, dinitial = torch.autograd.grad(final[1].sum(), (x, initial))         # (the second sequence's)
    ops.check_status()
    total = dx.double().sum(0) + dinitial.double()[1]
    # (what x gets from two sequences is added in its type: the first one's are zeros)
    assert float((total - 1).abs().max()) <= SLACK + torch.finfo(dtype).eps / 2 + 12 * 2.0 ** -24
    assert float(dinitial[0].abs().max()) == 0.0


@gpu
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 61), (BF, 64), (BF, 61)])
def test_steps_leave_a_state_that_equals_its_inputs(native, dtype, D):
    """Where less than half is taken, to the bit: the difference that is followed is zero."""
    value = (0.5 + torch.arange(D, device=DEV) % 7 / 8.0).to(dtype).expand(3, D).contiguous()
    gate = torch.linspace(0.1, 18.0, D, device=DEV).to(dtype).expand(3, D).contiguous()
    state = value.float().clone()
    for _ in range(50):
        assert torch.equal(gated_scan_step_(state, value, gate), value)
    assert torch.equal(state, value.float())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gate,length", [(-30.0, 3), (0.5, 3), (20.0, 3), (20.0, 5000)])
def test_infinite_states_and_far_ends(native, dtype, gate, length):
    """An infinite state stays infinite (as long as what is kept of it is more than zero), and an input and a state whose difference is above the largest
    number meet within their range."""
    D = 16
    top = 3e38
    x = torch.zeros(1, length, D, device=DEV, dtype=dtype)
    initial = torch.zeros(1, D, device=DEV)
    initial[0, :4] = torch.tensor([float("inf"), float("-inf"), top, -top], device=DEV)
    x[0, :, 2], x[0, :, 3] = -top, top
    x[0, 0, 4], x[0, 0, 5] = float("inf"), float("-inf")
    h, final = gated_scan(x, torch.full_like(x, gate), initial_state=initial, return_state=True)
    sign = torch.tensor([1.0, -1.0], device=DEV)
    for pair in (0, 4):
        assert torch.equal(h[0, :, pair:pair + 2].float(), (sign * float("inf")).expand(length, 2))
        assert torch.equal(final[0, pair:pair + 2], sign * float("inf"))
    assert bool(final[0, 2:4].isfinite().all()) and bool(h[0, :, 2:4].isfinite().all()) and bool((h[0, :, 6:] == 0).all())


@gpu
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF, 64), (BF, 61)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_a_bad_number_leaves_alone(native, dtype, D, bad):
    """A segment that meets an infinity or NaN is walked again: other channels, earlier rows and other sequences keep their bits, forward and backward."""
    B, length = 3, 5000
    g = torch.Generator(device=DEV).manual_seed(5)
    x, gate, dh = (torch.randn(B, length, D, generator=g, device=DEV).to(dtype) for _ in range(3))
    initial = torch.randn(B, D, generator=g, device=DEV)

    def run(x, initial, dh):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gate, initial)]
        h, final = gated_scan(*leaves[:2], initial_state=leaves[2], return_state=True)
        return [h.detach(), final.detach(), *torch.autograd.grad(h, leaves, dh)]
    want = run(x, initial, dh)
    at = 2345
    t = x.clone()
    t[1, at, 3] = bad
    h, final, dx, dgate, dinitial = run(t, initial, dh)
    keep = torch.ones(B, length, D, dtype=torch.bool, device=DEV)
    keep[1, at:, 3] = False
    assert torch.equal(h[keep], want[0][keep]) and torch.equal(dx, want[2]) and torch.equal(dinitial, want[4]) and torch.equal(dgate[keep], want[3][keep])
    assert not bool(h[1, at, 3].isfinite())
    t = dh.clone()
    t[1, at, 3] = bad
    h, final, dx, dgate, dinitial = run(x, initial, t)
    keep = torch.ones(B, length, D, dtype=torch.bool, device=DEV)
    keep[1, :at + 1, 3] = False
    assert torch.equal(h, want[0]) and torch.equal(dx[keep], want[2][keep]) and torch.equal(dgate[keep], want[3][keep])
    assert not bool(dx[1, at, 3].isfinite())
