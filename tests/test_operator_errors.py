"""Which error a failed operator raises, and with whose text.  The CUDA error is injected on the host before any launch."""
import pytest
import torch

from flame_b200 import CudaError, InvalidInput, _lib, _op

# without a GPU: a call that the injected error did not stop would run on addresses that are none
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="runs without a GPU")

FAKE = 1 << 20      # an aligned address that no call here touches
FAULT_KERNEL = 2    # FLAME_OFFLOAD_FAULT_KERNEL
WS = 1 << 24
# name, arguments it takes, and the place and value of one that it refuses
CALLS = [
    ("flame_dropout", [FAKE, None, FAKE, 8, 0, 0.5, 1, None, 0, None], 5, 1.5),
    ("flame_fp8_quant_2d", [FAKE, 4, 64, 64, FAKE, FAKE, 1, None, None, 64, None], 6, 7),
    ("flame_fp8_dequant_2d", [FAKE, 64, FAKE, 1, FAKE, 0, 4, 64, None], 3, 0),
    ("flame_fp8_product", [FAKE, 64, FAKE, 1, FAKE, 64, FAKE, 3, 1, FAKE, 16, 0, 8, 16, 64, None], 11, 7),
    ("flame_fp8_linear", [FAKE, 64, None, 0, None, FAKE, 64, None, 0, None, 0, FAKE, 8, 16, 64, FAKE, WS, None], 1, 63),
    ("flame_fp8_linear_backward", [FAKE, 16, FAKE, 64, FAKE, 64, None, 0, None, FAKE, FAKE, 8, 16, 64, FAKE, WS, None], 1, 15),
    ("flame_group_norm", [FAKE, None, None, FAKE, None, None, FAKE, 2, 10, 64, 8, 1e-5, 0, 0, FAKE, WS, None], 12, 5),
    ("flame_group_norm_backward", [FAKE, FAKE, None, None, FAKE, FAKE, None, None, 2, 10, 64, 8, 0, 0, FAKE, WS, None], 12, 5),
]


@pytest.mark.parametrize("name,args,at,bad", CALLS, ids=[c[0] for c in CALLS])
def test_a_cuda_error_does_not_keep_the_text_of_a_refusal(name, args, at, bad):
    lib = _lib.lib()
    refused = list(args)
    refused[at] = bad
    assert getattr(lib, name)(*refused) == 1 and _lib.last_error().startswith(name + ":")
    lib.flame_offload_inject_fault(FAULT_KERNEL, 1)
    try:
        assert getattr(lib, name)(*args) == 719
    finally:
        lib.flame_offload_inject_fault(0, 1)
    assert _lib.last_error().startswith(f"CUDA error in {name}: ") and "719" in _lib.last_error()


@pytest.mark.parametrize("code", [1, 719])
def test_it_is_raised_as_what_it_is(monkeypatch, code):
    """Also where CUDA's code is the one that refusals have."""
    name, args, at, bad = CALLS[0]
    lib = _lib.lib()
    refused = list(args)
    refused[at] = bad
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: None, raising=False)
    with pytest.raises(InvalidInput, match="flame_dropout: p must be"):
        _op.call(name, torch.device("cuda", 0), *refused[:-1])

    def failing(*a):
        lib.flame_offload_inject_fault(FAULT_KERNEL, 1)
        assert lib.flame_dropout(*a) == 719
        return code

    monkeypatch.setitem(_op._FUNCTIONS, name, failing)
    with pytest.raises(CudaError, match="CUDA error in flame_dropout"):
        _op.call(name, torch.device("cuda", 0), *args[:-1])
