"""A seed in device memory that changes between forward and backward is refused whatever holds the saved tensors.  No GPU: the launches are
stubbed out."""
import contextlib

import pytest
import torch

from flame_b200 import _op
from flame_b200 import checkpoint as ckpt
from flame_b200.dropout import dropout


@pytest.fixture
def launches(monkeypatch):
    seeds = []
    monkeypatch.setattr(_op, "on_gpu", lambda what, *tensors: torch.device("cpu"))
    monkeypatch.setattr(_op, "call", lambda name, device, x, residual, y, n, dtype, p, seed, seed_device, offset: seeds.append(seed_device))
    return seeds


def keep(t):
    return t


HOOKS = {
    "none": contextlib.nullcontext,
    "kept": lambda: torch.autograd.graph.saved_tensors_hooks(keep, keep),
    "copied": lambda: torch.autograd.graph.saved_tensors_hooks(torch.clone, keep),
}


@pytest.mark.parametrize("name", HOOKS)
def test_a_modified_seed_is_refused(launches, name):
    x, seed = torch.randn(16, requires_grad=True), torch.tensor([5])
    with HOOKS[name]():
        y = dropout(x, 0.5, seed=seed)
    seed.fill_(6)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()
    with HOOKS[name]():
        y = dropout(x, 0.5, seed=seed)
    y.sum().backward()
    assert launches == [seed.data_ptr()] * 3      # forward, forward, backward: all read the caller's tensor


def test_a_modified_seed_is_refused_where_the_block_is_recomputed(launches):
    x, seed = torch.randn(16, requires_grad=True), torch.tensor([5])
    y = ckpt.checkpoint([x], lambda t: dropout(t.sin(), 0.5, seed=seed).sin())
    seed.fill_(6)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()
