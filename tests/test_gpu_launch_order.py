"""What a recorded call's launches wait for.  A kernel that reads the call's inputs before it has waited for the kernel ahead of it is
started by that kernel, and that kernel by an ordinary launch: everything ahead of the call is complete when either runs."""
import ctypes

import pytest
import torch

from flame_b200.fp8_product import fp8_linear
from flame_b200.group_norm import group_norm, group_norm_fp8

pytestmark = pytest.mark.gpu


class EdgeData(ctypes.Structure):
    _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]


def chain(record):
    """The edges of a recorded run of kernels in the order of the launches: 'full' or 'early' (the kernel behind may start before the one
    ahead has ended)."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        kept = record()
    cuda = ctypes.CDLL("libcuda.so.1")
    cuda.cuGraphGetEdges_v2.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]
    handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert cuda.cuGraphGetEdges_v2(handle, None, None, None, ctypes.byref(count)) in (0, 911)      # 911: there are edges that are not full
    sources, targets, data = (ctypes.c_void_p * count.value)(), (ctypes.c_void_p * count.value)(), (EdgeData * count.value)()
    assert cuda.cuGraphGetEdges_v2(handle, sources, targets, data, ctypes.byref(count)) == 0
    behind = {sources[i]: (targets[i], "early" if data[i].type else "full") for i in range(count.value)}
    assert len(behind) == count.value
    at, = set(sources) - set(targets)
    kinds = []
    while at in behind:
        at, kind = behind[at]
        kinds.append(kind)
    del kept
    return kinds


def test_group_norm(cuda_device):
    w = torch.ones(640, device=cuda_device)
    for positions, launches in ((1000, 2), (200000, 3)):       # three: the parts are joined by a launch of their own
        x = torch.randn(1, positions, 640, device=cuda_device).to(torch.bfloat16).requires_grad_(True)
        dy = torch.randn_like(x)
        group_norm(x, 32, w)
        for forward in (lambda: group_norm(x.detach(), 32, w), lambda: group_norm_fp8(x.detach(), 32, w)):
            forward()
            torch.cuda.synchronize()

            def record():
                x.detach().mul_(1.5)
                return forward()

            assert chain(record) == ["full"] + ["early"] * (launches - 1)

        def step():
            y = group_norm(x, 32, w)
            z = y.detach() * 2
            return z, torch.autograd.grad(y, x, dy * z)

        step()
        torch.cuda.synchronize()
        kinds = chain(step)
        assert kinds == ["early"] * (launches - 1) + ["full"] * 3 + ["early"] * (launches - 1)


def test_linear_layer(cuda_device):
    x, w, dy = (torch.randn(s, device=cuda_device).to(torch.bfloat16) for s in ((1000, 256), (512, 256), (1000, 512)))
    x.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        y = fp8_linear(x, w)
        return torch.autograd.grad(y, (x, w), dy * y.detach())

    step()
    torch.cuda.synchronize()
    # quantiser, product, multiplication, quantiser, the input gradient's product, and the weight gradient's, which begins early
    kinds = chain(step)
    assert kinds[0] == "early" and kinds[-2:] == ["full", "early"]
