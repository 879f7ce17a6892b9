"""Arguments of another kind than documented are refused by name.  No GPU: nothing is launched."""
import pytest
import torch

from flame_b200 import InvalidInput, _op
from flame_b200.fp8_product import fp8_linear


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    monkeypatch.setattr(_op, "on_gpu", lambda what, *tensors: torch.device("cpu"))


def test_linear_layer():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for weight in (None, [1.0], "w"):
        with pytest.raises(InvalidInput, match="expected a tensor or Fp8Blocks as weight"):
            fp8_linear(x, weight)
    for codes in (x, "rows", (x, x)):
        with pytest.raises(InvalidInput, match="codes are Fp8Blocks"):
            fp8_linear(x, x, codes=codes)
