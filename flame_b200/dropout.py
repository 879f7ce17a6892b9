"""Dropout whose mask is never stored.

The mask is a function of (seed, offset, element index), so there is nothing to save, to offload or to recompute state for: the
backward pass draws the same numbers again, and so does a forward pass that ``checkpoint`` runs a second time.  The caller gives
each dropout of a model an ``offset`` of its own and changes the ``seed`` from step to step::

    h = dropout(h, 0.1, seed=step_seed, offset=2 * layer)
    x = dropout(h, 0.1, seed=step_seed, offset=2 * layer + 1, residual=x)     # x + dropout(h), one pass

A step recorded in a CUDA graph takes ``seed`` as an int64 tensor of one element on the GPU, which is read when the kernel runs:
write the next seed into it between replays.  Where backward runs outside that graph, leave the tensor alone until it has run
(a seed that was modified is refused).

csrc/dropout.cu defines the numbers: Philox 4x32-10, 32 bits for each element.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _op
from .errors import InvalidInput


def _launch(x, residual, p, seed, offset):
    y = torch.empty_like(x)
    device_seed = seed if isinstance(seed, torch.Tensor) else None
    _op.call("flame_dropout", x.device, x.data_ptr(), _op.ptr(residual), y.data_ptr(), x.numel(), _op.DTYPE[x.dtype], p,
             0 if device_seed is not None else seed, _op.ptr(device_seed), offset)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.p, ctx.offset = p, offset
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        if ctx.seed is None:      # autograd does not look at the version of a tensor that goes through saved-tensor hooks
            ctx.seed_tensor, ctx.seed_version = seed, seed._version
        return _launch(x, residual, p, seed, offset)

    @_op.first_order
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            seed = ctx.seed
            if seed is None:
                seed = ctx.seed_tensor
                if seed._version != ctx.seed_version:
                    raise RuntimeError("dropout: the seed tensor was modified between forward and backward")
            dx = _launch(dy.contiguous(), None, ctx.p, seed, ctx.offset)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, *, seed: Union[int, torch.Tensor], offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x / (1 - p)`` where an element is kept and 0 where it is dropped, plus ``residual``; BF16 or F32, contiguous.

    ``p`` is exact to 2^-32.  A dropped element is 0 whatever it was, infinities and NaN included."""
    _op.on_gpu("dropout", x, residual)
    if x.dtype not in _op.DTYPE:
        raise InvalidInput("dropout: BF16 or F32 tensors")
    if not x.is_contiguous():
        raise InvalidInput("dropout: x must be contiguous")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise InvalidInput(f"dropout: p must be in [0, 1], got {p}")
    if not (isinstance(offset, int) and 0 <= offset < 1 << 64):
        raise InvalidInput("dropout: offset must be an integer in [0, 2^64)")
    if isinstance(seed, torch.Tensor):
        if not (seed.device == x.device and seed.dtype == torch.int64 and seed.numel() == 1):
            raise InvalidInput("dropout: a seed tensor holds one int64 on the device of x")
    elif not (isinstance(seed, int) and 0 <= seed < 1 << 64):
        raise InvalidInput("dropout: seed must be an integer in [0, 2^64) or a tensor")
    if residual is not None and not (residual.dtype == x.dtype and residual.shape == x.shape and residual.is_contiguous()):
        raise InvalidInput("dropout: residual must be contiguous, with the type and shape of x")
    if not _op.recorded(x, residual):
        return _launch(x, residual, p, seed, offset)
    return _Dropout.apply(x, residual, p, seed, offset)
