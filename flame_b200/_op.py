"""What the operator modules share: argument checks, the device a call runs on, and the translation of the library's codes."""
from __future__ import annotations

import torch

from . import _lib
from .errors import CudaError, InvalidInput

DTYPE = {torch.bfloat16: 0, torch.float32: 1}     # FLAME_OFFLOAD_DTYPE_*


def need(cond: bool, message: str, error=InvalidInput) -> None:
    if not cond:
        raise error(message)


def on_gpu(what: str, *tensors) -> torch.device:
    """The one GPU that all the tensors (None is skipped) are on."""
    device = None
    for t in tensors:
        if t is None:
            continue
        need(isinstance(t, torch.Tensor), f"{what}: expected a tensor, got {type(t).__name__}")
        need(t.is_cuda, f"{what}: the tensors must be on the GPU")
        need(device is None or t.device == device, f"{what}: the tensors must be on one device")
        device = t.device
    return device


def call(name: str, device: torch.device, *args) -> None:
    """`name`(*args, stream) on the current stream of `device`, whichever device is the current one."""
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc == 1:
        raise InvalidInput(_lib.last_error() or f"{name}: invalid argument")
    if rc != 0:
        raise CudaError(f"{name} failed ({rc})")


def ptr(t):
    return None if t is None else t.data_ptr()
