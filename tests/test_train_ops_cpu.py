"""What the operators around the layer do on the host, without a GPU: argument checks, and norms over a process group."""
import os
import sys
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from streamep_b200 import _ext
from streamep_b200.ops import adamw_step_, clip_grad_norm_, grad_norm, linear_cross_entropy


def test_refused_before_anything_native():
    x, w, y = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="average")
    with pytest.raises(ValueError, match="shape"):
        linear_cross_entropy(x, w, y[:3])
    for kw, what in ((dict(max_norm=1.0), "norm"), (dict(skip_nonfinite=True), "norm"), (dict(norm=torch.ones(()), max_norm=-1.0), "negative"), (dict(masters=[]), "masters")):
        with pytest.raises(ValueError, match=what):
            adamw_step_([x], [x], [x], [x], step=1, lr=0.1, **kw)


def test_refused_by_the_native_side_without_a_gpu():
    for f in (lambda t: grad_norm([t]), lambda t: clip_grad_norm_([t], 1.0)):
        with pytest.raises(ValueError, match="CUDA"):
            f(torch.ones(4))
    with pytest.raises(ValueError, match="negative"):
        clip_grad_norm_([torch.ones(4)], -1.0)
    with pytest.raises(ValueError, match="not a tensor"):
        grad_norm([1.0])


class FakeNative:
    """The native calls on the CPU, by their definitions."""

    @staticmethod
    def list_norm(ts):
        s = sum((t.double().square().sum() for t in ts), torch.zeros((), dtype=torch.float64))
        return s.sqrt().float(), s

    @staticmethod
    def list_scale(ts, norm, max_norm):
        for t in ts:
            t.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))


def _rank(rank, world, store, out):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world)
    _ext.load = lambda: FakeNative
    shared, mine = [torch.full((10,), 2.0), torch.full((3,), -1.0)], [torch.full((7,), float(rank + 1))]
    if rank == 1:                     # a rank without sharded gradients takes part all the same
        alone = grad_norm(shared, sharded=[], group=dist.group.WORLD)
    else:
        alone = grad_norm(shared, sharded=mine, group=dist.group.WORLD)
    assert abs(float(alone) - (40.0 + 3.0 + 7.0) ** 0.5) < 1e-5
    norm = grad_norm(shared, sharded=mine, group=dist.group.WORLD)
    clipped = clip_grad_norm_(shared, 3.0, sharded=mine, group=dist.group.WORLD)
    torch.save((norm, clipped, shared, mine), f"{out}.{rank}")
    dist.destroy_process_group()


def test_norm_over_a_group():
    """Replicated gradients count once, sharded ones on every rank."""
    with tempfile.TemporaryDirectory() as d:
        out = os.path.join(d, "out")
        mp.spawn(_rank, args=(2, os.path.join(d, "store"), out), nprocs=2)
        want = (40.0 + 3.0 + 7.0 * 1 + 7.0 * 4) ** 0.5
        for rank in range(2):
            norm, clipped, shared, mine = torch.load(f"{out}.{rank}")
            assert abs(float(norm) - want) < 1e-5 and abs(float(clipped) - want) < 1e-5
            f = 3.0 / (want + 1e-6)
            torch.testing.assert_close(shared[0], torch.full((10,), 2.0 * f))
            torch.testing.assert_close(mine[0], torch.full((7,), (rank + 1) * f))
