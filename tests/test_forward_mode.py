"""Forward-mode derivatives of the operators are refused, not dropped.  No GPU: the launches are stubbed out."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from flame_b200 import _op
from flame_b200.dropout import dropout
from flame_b200.fp8_product import Fp8Blocks, fp8_linear
from flame_b200.group_norm import group_norm, group_norm_fp8


@pytest.fixture
def launches(monkeypatch):
    """Names of the library's calls, none of which runs."""
    names = []
    monkeypatch.setattr(_op, "on_gpu", lambda what, *tensors: torch.device("cpu"))
    monkeypatch.setattr(_op, "call", lambda name, *args: names.append(name))
    monkeypatch.setattr(_op, "function", lambda name: lambda *args: 64)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    return names


def bf(*shape):
    return torch.randn(*shape).to(torch.bfloat16)


X, W, V = (4, 128), (256, 128), (128,)
FROZEN = lambda: Fp8Blocks(torch.zeros(W, dtype=torch.uint8), torch.ones(2, 1), "tiles")  # noqa: E731
CALLS = {
    "linear, x": (X, lambda t: fp8_linear(t, bf(*W))),
    "linear, weight": (W, lambda t: fp8_linear(bf(*X), t)),
    "linear, frozen weight": (X, lambda t: fp8_linear(t, FROZEN())),
    "group norm, x": (X, lambda t: group_norm(t, 8)),
    "group norm, weight": (V, lambda t: group_norm(bf(*X), 8, t)),
    "group norm, bias": (V, lambda t: group_norm(bf(*X), 8, None, t)),
    "group norm with codes": (X, lambda t: group_norm_fp8(t, 8)[0]),
    "dropout, x": (X, lambda t: dropout(t, 0.5, seed=1)),
    "dropout, residual": (X, lambda t: dropout(bf(*X), 0.5, seed=1, residual=t)),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(launches, name, grad):
    shape, f = CALLS[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
            f(forward_ad.make_dual(bf(*shape), bf(*shape)))
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
            f(forward_ad.make_dual(bf(*shape).requires_grad_(True), bf(*shape)))


@pytest.mark.parametrize("name", CALLS)
def test_a_level_without_tangents_changes_nothing(launches, name):
    shape, f = CALLS[name]
    for level in (contextlib.nullcontext(), forward_ad.dual_level()):
        with level:
            assert not f(bf(*shape)).requires_grad and f(bf(*shape).requires_grad_(True)).requires_grad
    assert len(launches) == 4
