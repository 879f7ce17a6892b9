"""The operators' refusals that need no GPU: bad arguments come back as an error code and a text before any CUDA call."""
import pytest
import torch

from flame_b200 import InvalidInput, _lib
from flame_b200.dropout import dropout
from flame_b200.fp8_product import Fp8Blocks, fp8_linear, quantize_fp8
from flame_b200.group_norm import group_norm

FAKE = 1 << 20      # an aligned address that no refused call may touch


def refused(text, name, *args):
    lib = _lib.lib()
    assert getattr(lib, name)(*args) == 1
    assert text in _lib.last_error(), _lib.last_error()


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: quantize_fp8(x), lambda: fp8_linear(x, x), lambda: group_norm(x, 8), lambda: dropout(x, 0.5, seed=1),
              lambda: Fp8Blocks(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1), "rows")):
        with pytest.raises(InvalidInput, match="on the GPU"):
            f()


def test_what_is_no_tensor_is_refused():
    for f in (lambda: quantize_fp8(None), lambda: group_norm(None, 8), lambda: dropout(None, 0.5, seed=1), lambda: fp8_linear([1.0], None)):
        with pytest.raises(InvalidInput, match="expected a tensor"):
            f()


def test_quantiser_entry():
    ok = [FAKE, 4, 64, 64, FAKE, FAKE, 1, None, None, 64, None]
    for at, value, text in ((6, 7, "blocks must be"), (6, 0, "nothing to make"), (3, 63, "stride"), (9, 48, "stride"), (9, 72, "stride"), (0, None, "null"), (4, None, "null"),
                            (4, FAKE + 8, "misaligned"), (0, FAKE + 1, "misaligned"), (1, 1 << 40, "too large"), (2, 1 << 40, "too large")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_fp8_quant_2d", *bad)
    refused("one call", "flame_fp8_quant_2d", FAKE, 4, 64, 64, FAKE, FAKE, 3, FAKE, FAKE, 64, None)
    refused("null", "flame_fp8_quant_2d", FAKE, 4, 64, 64, FAKE, FAKE, 1, FAKE, None, 64, None)
    assert _lib.lib().flame_fp8_quant_2d(None, 0, 64, 64, None, None, 1, None, None, 64, None) == 0


def test_dequantiser_entry():
    ok = [FAKE, 64, FAKE, 1, FAKE, 0, 4, 64, None]
    for at, value, text in ((3, 0, "blocks"), (5, 2, "BF16 or F32"), (1, 63, "stride"), (0, None, "null"), (0, FAKE + 4, "misaligned"), (6, 1 << 40, "too large")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_fp8_dequant_2d", *bad)
    assert _lib.lib().flame_fp8_dequant_2d(None, 64, None, 1, None, 0, 0, 64, None) == 0


def test_product_entry():
    ok = [FAKE, 64, FAKE, 1, FAKE, 64, FAKE, 3, 1, FAKE, 16, 0, 8, 16, 64, None]
    for at, value, text in ((3, 2, "contraction"), (7, 2, "contraction"), (8, 0, "stride"), (1, 48, "stride"), (5, 68, "stride"), (10, 15, "stride"), (11, 7, "BF16 or F32"),
                            (9, None, "output"), (0, None, "null"), (6, None, "null"), (4, FAKE + 8, "misaligned"), (12, 1 << 33, "too large"), (14, 1 << 33, "too large")):
        bad = list(ok)
        bad[at] = value
        if at == 8:
            bad[13] = 80          # b read as [K, N]: its rows of 80 do not fit a stride of 64
        refused(text, "flame_fp8_product", *bad)
    lib = _lib.lib()
    assert lib.flame_fp8_product(None, 64, None, 1, None, 64, None, 3, 1, None, 16, 0, 0, 16, 64, None) == 0


def test_linear_entries():
    lib = _lib.lib()
    assert lib.flame_fp8_linear_workspace_bytes(1 << 40, 1, 1, 0) == 0
    size = lib.flame_fp8_linear_workspace_bytes(8, 16, 64, 2)
    ok = [FAKE, 64, None, 0, None, FAKE, 64, None, 0, None, 0, FAKE, 8, 16, 64, FAKE, size, None]
    for at, value, text in ((0, None, "null"), (1, 63, "stride"), (6, 60, "stride"), (11, None, "null"), (11, FAKE + 1, "misaligned"), (15, FAKE + 16, "workspace"), (16, size - 1, "workspace"),
                            (12, 1 << 40, "too large"), (2, FAKE, "stride")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_fp8_linear", *bad)
    refused("tiles or rows", "flame_fp8_linear", FAKE, 64, None, 0, None, None, 0, FAKE, 64, FAKE, 2, FAKE, 8, 16, 64, FAKE, size, None)
    refused("null", "flame_fp8_linear", FAKE, 64, None, 0, None, None, 0, FAKE, 64, None, 3, FAKE, 8, 16, 64, FAKE, size, None)
    size = lib.flame_fp8_linear_workspace_bytes(8, 16, 64, 3)
    ok = [FAKE, 16, FAKE, 64, FAKE, 64, None, 0, None, FAKE, FAKE, 8, 16, 64, FAKE, size, None]
    for at, value, text in ((0, None, "null"), (1, 15, "stride"), (2, None, "null"), (3, 63, "stride"), (5, 63, "stride"), (9, FAKE + 1, "misaligned"), (15, size - 1, "workspace")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_fp8_linear_backward", *bad)
    assert lib.flame_fp8_linear(None, 64, None, 0, None, None, 0, None, 64, None, 3, None, 0, 16, 64, None, 0, None) == 0


def test_group_norm_entries():
    lib = _lib.lib()
    assert lib.flame_group_norm_workspace_bytes(2, 10, 64, 7, 0) == 0 and "multiple" in _lib.last_error()
    size = lib.flame_group_norm_workspace_bytes(2, 10, 64, 8, 0)
    assert size > 0
    ok = [FAKE, None, None, FAKE, None, None, FAKE, 2, 10, 64, 8, 1e-5, 0, 0, FAKE, size, None]
    for at, value, text in ((10, 0, "multiple"), (9, 1 << 20, "channels"), (7, 1 << 20, "samples"), (12, 5, "activation"), (13, 5, "BF16 or F32"), (0, None, "null"), (14, None, "null"),
                            (15, size - 4, "workspace"), (14, FAKE + 4, "misaligned"), (4, FAKE, "codes")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_group_norm", *bad)
    size = lib.flame_group_norm_workspace_bytes(2, 10, 64, 8, 1)
    ok = [FAKE, FAKE, None, None, FAKE, FAKE, None, None, 2, 10, 64, 8, 0, 0, FAKE, size, None]
    for at, value, text in ((1, None, "null"), (5, None, "null"), (15, 0, "workspace"), (12, 2, "activation"), (11, 3, "multiple")):
        bad = list(ok)
        bad[at] = value
        refused(text, "flame_group_norm_backward", *bad)
    assert lib.flame_group_norm(None, None, None, None, None, None, None, 0, 10, 64, 8, 1e-5, 0, 0, None, 0, None) == 0


def test_group_norm_alignment():
    """Pairs of statistics are written at once, parameters read as what they are."""
    lib = _lib.lib()
    size = lib.flame_group_norm_workspace_bytes(2, 10, 128, 8, 0)
    ok = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 10, 128, 8, 1e-5, 0, 1, FAKE, size, None]
    for at, value in ((0, FAKE + 1), (1, FAKE + 2), (2, FAKE + 2), (3, FAKE + 1), (5, FAKE + 2), (6, FAKE + 4)):
        bad = list(ok)
        bad[at] = value
        refused("misaligned", "flame_group_norm", *bad)
    size = lib.flame_group_norm_workspace_bytes(2, 10, 128, 8, 1)
    ok = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 10, 128, 8, 0, 1, FAKE, size, None]
    for at, value in ((0, FAKE + 1), (1, FAKE + 1), (2, FAKE + 2), (3, FAKE + 2), (4, FAKE + 4), (5, FAKE + 1), (6, FAKE + 2), (7, FAKE + 2)):
        bad = list(ok)
        bad[at] = value
        refused("misaligned", "flame_group_norm_backward", *bad)


def test_dropout_entry():
    for args, text in (((FAKE, None, FAKE, 8, 0, 1.5, 1, None, 0, None), "p must be"), ((FAKE, None, FAKE, 8, 0, float("nan"), 1, None, 0, None), "p must be"),
                       ((FAKE, None, FAKE, 8, 3, 0.5, 1, None, 0, None), "dtype"), ((None, None, FAKE, 8, 0, 0.5, 1, None, 0, None), "null"),
                       ((FAKE + 1, None, FAKE, 8, 0, 0.5, 1, None, 0, None), "misaligned"), ((FAKE, FAKE + 2, FAKE, 8, 1, 0.5, 1, None, 0, None), "misaligned"),
                       ((FAKE, None, FAKE, 8, 0, 0.5, 1, FAKE + 4, 0, None), "misaligned")):
        refused(text, "flame_dropout", *args)
    assert _lib.lib().flame_dropout(None, None, None, 0, 0, 0.5, 1, None, 0, None) == 0
