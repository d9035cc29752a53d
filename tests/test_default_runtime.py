"""Calls without a buffer: a runtime for each device, and a public way to ask what they reported."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from streamep_b200 import StreamEPError, StreamEPTimeout, _ext, ops
from streamep_b200.ops import grouped_gemm as gg


class FakeRuntime:
    device, message = None, ""

    def __init__(self, *args):
        self.device = torch.cuda.current_device()

    def get_local_base_ptr(self):
        return 0

    def sync_local(self, pointers):
        assert torch.cuda.current_device() == self.device

    def poll_status(self, reset):
        assert torch.cuda.current_device() == self.device and reset
        message, self.message = self.message, ""
        return message


@pytest.fixture
def two_devices(monkeypatch):
    current = [0]

    @contextlib.contextmanager
    def on(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(_ext, "load", lambda: SimpleNamespace(Runtime=FakeRuntime, MAX_EXPERTS=1024))
    monkeypatch.setattr(gg, "_default_runtimes", {})


def test_a_runtime_for_each_device(two_devices):
    ops.check_status()                                        # nothing was called, nothing is made
    first, second = gg.default_runtime(), gg.default_runtime(torch.device("cuda", 1))
    assert (first.device, second.device) == (0, 1)
    assert gg._rt(None, torch.device("cuda", 1)) is second and gg._rt(None) is first and gg.default_runtime(torch.device("cuda")) is first
    second.message = "tile gate timeout (code 3)"
    ops.check_status()
    with pytest.raises(StreamEPTimeout, match="gate"):
        ops.check_status("cuda:1")
    first.message = "target outside the vocabulary (where = token)"
    with pytest.raises(StreamEPError, match="outside the vocabulary"):
        ops.check_status(torch.device("cuda", 0))
    ops.check_status()
    ops.check_status(torch.device("cuda", 1))


def test_the_loss_takes_the_runtime_of_its_tensors(two_devices):
    asked = []
    with pytest.MonkeyPatch.context() as m:
        m.setattr("streamep_b200.ops.linear_loss._rt", lambda buffer, device=None: asked.append(device) or SimpleNamespace(linear_loss=lambda *a: torch.zeros(())))
        x = SimpleNamespace(dim=lambda: 2, shape=(2, 8), is_cuda=True, device=torch.device("cuda", 1))
        ops.linear_cross_entropy(x, None, torch.zeros(2, dtype=torch.int64))
    assert asked == [torch.device("cuda", 1)]
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_cross_entropy(torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(2, dtype=torch.int64))


@pytest.mark.gpu
def test_bad_target_without_a_buffer(native):
    x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(100, 64, device="cuda").bfloat16()
    y = torch.zeros(40, dtype=torch.int64, device="cuda")
    ops.linear_cross_entropy(x, w, y)
    ops.check_status()
    y[3] = 100
    assert torch.isnan(ops.linear_cross_entropy(x, w, y))
    with pytest.raises(StreamEPError, match="outside the vocabulary"):
        ops.check_status()
    ops.check_status()
