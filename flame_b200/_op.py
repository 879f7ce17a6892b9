"""What the operator modules share: the device a call runs on, and the translation of the library's codes.

These modules run once for every layer and step, and at small sizes the host decides how long that takes: messages are built only
when something is refused, and a call that nobody differentiates leaves no autograd node.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .errors import CudaError, InvalidInput

DTYPE = {torch.bfloat16: 0, torch.float32: 1}     # FLAME_OFFLOAD_DTYPE_*

_FUNCTIONS: dict = {}


def on_gpu(what: str, *tensors) -> torch.device:
    """The one GPU that all the tensors (None is skipped) are on."""
    index = first = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise InvalidInput(f"{what}: expected a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise InvalidInput(f"{what}: the tensors must be on the GPU")
        if index is None:
            index, first = t.get_device(), t
        elif t.get_device() != index:
            raise InvalidInput(f"{what}: the tensors must be on one device")
    if first is None:
        raise InvalidInput(f"{what}: expected a tensor, got None")
    return first.device


def function(name: str):
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.lib(), name)
    return fn


def call(name: str, device: torch.device, *args) -> None:
    """`name`(*args, stream) on the current stream of `device`, whichever device is the current one."""
    fn = function(name)
    index = device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        text = _lib.last_error()
        if rc == 1 and text.startswith(name + ":"):      # an error of CUDA's has a text that begins otherwise
            raise InvalidInput(text)
        raise CudaError(text or f"{name} failed ({rc})")


def workspace(like, size: int):
    """`size` bytes on the device of `like`, a BF16 tensor (which is quicker than to name type and device)."""
    return like.new_empty((size + 1) // 2)


def ptr(t):
    return None if t is None else t.data_ptr()


def recorded(*tensors) -> bool:
    """Whether autograd records a call on these tensors (None is skipped).  A tensor with a forward-mode tangent counts: the recorded form
    refuses it, where a bare launch would drop the tangent."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def first_order(f):
    """A backward that gives first derivatives: a second one is refused by autograd.  The wrapper that says so costs a third of a small
    call's time, so only a backward pass that is itself recorded (``create_graph=True``) goes through it."""
    recorded_form = once_differentiable(f)

    @functools.wraps(f)
    def backward(ctx, *grads):
        return recorded_form(ctx, *grads) if torch.is_grad_enabled() else f(ctx, *grads)

    return staticmethod(backward)
