"""The norm over a group with an empty list: its zero stands where the other list's sum stands, not on the device that is current."""
import pytest
import torch

from streamep_b200 import _ext
from streamep_b200.ops import clip_grad_norm_, grad_norm


class Group:
    def size(self):
        return 2


class Native:
    """Sums stand with the tensors ("cpu"); of nothing, on the current device ("meta" here)."""

    @staticmethod
    def list_norm(ts):
        if not ts:
            return torch.zeros((), device="meta"), torch.zeros((), dtype=torch.float64, device="meta")
        s = sum(t.double().square().sum() for t in ts)
        return s.sqrt().float(), s

    @staticmethod
    def list_scale(ts, norm, max_norm):
        assert all(norm.device == t.device for t in ts)


@pytest.mark.parametrize("grads,sharded", [([3.0], []), ([], [4.0]), ([3.0], [4.0])])
def test_device_of_an_empty_list(monkeypatch, grads, sharded):
    monkeypatch.setattr(_ext, "load", lambda: Native)
    reduced = []
    monkeypatch.setattr(torch.distributed, "all_reduce", lambda t, group=None: reduced.append(t.device.type))
    lists = [torch.tensor([v]) for v in grads], [torch.tensor([v]) for v in sharded]
    want = sum(v * v for v in grads + sharded) ** 0.5
    for call in (lambda: grad_norm(lists[0], sharded=lists[1], group=Group()), lambda: clip_grad_norm_(lists[0], 1.0, sharded=lists[1], group=Group())):
        norm = call()
        assert norm.device.type == "cpu" and norm.dtype == torch.float32 and float(norm) == want
    assert reduced == ["cpu", "cpu"]                        # every rank takes part, also one without sharded gradients
