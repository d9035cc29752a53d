"""``launch_count()`` of a call is the number of kernels that it launches: those of a captured call, counted in the graph."""
import pytest
import torch

from streamep_b200.models.moe_layer import make_buffer
from streamep_b200.ops import balanced_router, gated_scan

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def kernels_of(call, buf):
    """{"counted": ..., "launched": ...} of call(), which is made once before."""
    runtime = pytest.importorskip("cuda.bindings.runtime")

    def checked(result):
        assert result[0] == runtime.cudaError_t.cudaSuccess
        return result[1:]
    held = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = buf.runtime.launch_count()
    with torch.cuda.graph(graph):
        held = call()
    counted = buf.runtime.launch_count() - before
    raw = runtime.cudaGraph_t(graph.raw_cuda_graph())
    _, n = checked(runtime.cudaGraphGetNodes(raw))
    nodes, _ = checked(runtime.cudaGraphGetNodes(raw, n))
    kinds = [checked(runtime.cudaGraphNodeGetType(node))[0] for node in nodes]
    del held
    return {"counted": counted, "launched": kinds.count(runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel)}


# one segment a sequence, segments within a block, over blocks; odd channels
@pytest.mark.parametrize("shape", [(2000, 8, 64), (4, 200, 64), (1, 9000, 64), (2, 3000, 33)])
def test_recurrence(native, shape):
    buf = make_buffer(None, 64, 64, 2, 4)
    x, gate, dh = (torch.randn(shape, device=DEV).to(BF) for _ in range(3))
    leaves = [x.requires_grad_(True), gate.requires_grad_(True)]
    with torch.no_grad():
        forward = kernels_of(lambda: gated_scan(x, gate, buffer=buf), buf)
    both = kernels_of(lambda: torch.autograd.grad(gated_scan(*leaves, buffer=buf), leaves, dh), buf)
    assert forward["counted"] == forward["launched"] and both["counted"] == both["launched"], (forward, both)
    assert forward["launched"] == (2 if shape[1] >= 3000 else 1) and both["launched"] == 2 * forward["launched"]


# tokens in one part of dW and in several; gradients of x alone, of w alone
@pytest.mark.parametrize("T,H,E", [(100, 256, 8), (8192, 512, 64), (3000, 1024, 200)])
def test_routing(native, T, H, E):
    buf = make_buffer(None, 64, 64, 2, 4)
    x, w = torch.randn(T, H, device=DEV).to(BF), (torch.randn(E, H, device=DEV) * 0.02).to(BF)
    up = torch.randn(T, 2, device=DEV)
    with torch.no_grad():
        got = kernels_of(lambda: balanced_router(x, w, 2, buffer=buf), buf)
        assert got == {"counted": 2, "launched": 2}
    for wants in ((True, True), (True, False), (False, True)):
        leaves = [t.detach().requires_grad_(g) for t, g in zip((x, w), wants)]
        picked = [t for t in leaves if t.requires_grad]
        got = kernels_of(lambda: torch.autograd.grad(balanced_router(*leaves, 2, buffer=buf).topk_weights, picked, up), buf)
        assert got["counted"] == got["launched"], (wants, got)
        assert got["launched"] == 3 + (0 if not wants[1] else 1 if T == 100 else 2)
