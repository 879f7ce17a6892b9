"""Waits of the FP8 product that give up: who is told."""
import contextlib
import ctypes

import pytest
import torch

from flame_b200 import CudaError, _lib, _op, dit_workload, fp8_product


def counting(monkeypatch, counts, rc=0):
    """The library's counter, reading `counts` one after the other."""
    left = list(counts)

    def entry(out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_uint))[0] = left.pop(0)
        return rc

    monkeypatch.setitem(_op._FUNCTIONS, "flame_fp8_product_faults", entry)
    monkeypatch.setattr(fp8_product, "_seen_faults", {})
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def test_new_faults_are_raised_once(monkeypatch):
    counting(monkeypatch, [0, 3, 3, 4])
    fp8_product.check_faults()
    with pytest.raises(CudaError, match="3 warps on GPU 0"):
        fp8_product.check_faults(torch.device("cuda", 0))
    fp8_product.check_faults("cuda")
    with pytest.raises(CudaError, match="1 warps"):
        fp8_product.check_faults()


def test_devices_are_counted_apart(monkeypatch):
    counting(monkeypatch, [2, 2, 2])
    for index in (0, 1):
        with pytest.raises(CudaError, match=f"2 warps on GPU {index}"):
            fp8_product.check_faults(torch.device("cuda", index))
    fp8_product.check_faults("cuda:1")


def test_an_error_of_the_library_is_raised(monkeypatch):
    counting(monkeypatch, [0], rc=719)
    with pytest.raises(CudaError, match="719"):
        fp8_product.check_faults()


def test_the_workloads_steps_are_checked(monkeypatch):
    """The timed steps end with a wait for the device; the check stands behind it where the products are in FP8."""
    class Timer:
        def record(self): pass
        def elapsed_time(self, other): return 1.0

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.ones(4))

        def forward(self, x, cos, sin):
            return x * self.w

    model = Model()
    for name, value in (("synchronize", lambda: None), ("reset_peak_memory_stats", lambda: None), ("max_memory_allocated", lambda: 0),
                        ("memory_allocated", lambda: 0), ("Event", lambda enable_timing: Timer())):
        monkeypatch.setattr(torch.cuda, name, value)
    args = (model, torch.optim.SGD(model.parameters(), lr=0.1), torch.ones(4), None, None, 1, 1)
    counting(monkeypatch, [1])
    dit_workload._time_steps(*args)
    monkeypatch.setattr(dit_workload, "FP8_LINEARS", True)
    with pytest.raises(CudaError, match="gave up"):
        dit_workload._time_steps(*args)


def test_null_count_is_refused():
    assert _lib.lib().flame_fp8_product_faults(None) == 1 and "flame_fp8_product_faults: null" in _lib.last_error()


@pytest.mark.gpu
def test_the_check_waits_for_streams_of_their_own(cuda_device):
    """A stream that does not synchronise with the default one: the counter is read when its products have run, too."""
    x = torch.randn(4096, 4096, device=cuda_device).to(torch.bfloat16)
    w = fp8_product.quantize_fp8(x, "tiles")
    fp8_product.fp8_linear(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(300):
            fp8_product.fp8_linear(x, w)
    fp8_product.check_faults(cuda_device)
    assert side.query()
