"""Group norm with an activation on channels-last tensors, beside the RMSNorm producer.

``x`` is ``[batch, positions..., channels]``, BF16 and contiguous (a ``[B, C, H, W]`` tensor in channels-last memory is
``x.permute(0, 2, 3, 1)``).  The activation is part of both passes: backward needs ``x`` and two floats for each sample and group,
so a block saves one tensor for the norm and its activation, and a pool can offload it.
``group_norm_fp8`` also writes the FP8 codes of its output, the left operand of ``fp8_product.fp8_linear``.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import _op
from .errors import InvalidInput
from .fp8_product import Fp8Blocks

_ACTIVATIONS = {None: 0, "none": 0, "silu": 1}     # FLAME_ACTIVATION_*


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device_index, b, l, c, groups, backward) -> int:
    with torch.cuda.device(device_index):
        return max(_op.function("flame_group_norm_workspace_bytes")(b, l, c, groups, backward), 16)


def _sizes(x):
    shape = x.shape
    b, c = shape[0], shape[-1]
    if len(shape) == 3:
        return b, shape[1], c
    l = 1
    for n in shape[1:-1]:
        l *= n
    return b, l, c


def _forward(x, weight, bias, groups, eps, activation, codes_wanted, stats_wanted):
    device = x.device
    b, l, c = _sizes(x)
    y = torch.empty_like(x)
    stats = torch.empty(b, groups, 2, dtype=torch.float32, device=device) if stats_wanted else None
    codes = scales = None
    if codes_wanted:
        codes = torch.empty(b * l, c, dtype=torch.uint8, device=device)
        scales = torch.empty(b * l, c // 128, dtype=torch.float32, device=device)
    size = _workspace_bytes(device.index, b, l, c, groups, 0)
    # statistics that nobody reads again lie behind the workspace: an allocation costs a tenth of a small call's time
    ws = _op.workspace(x, size if stats_wanted else size + 8 * b * groups)
    at = ws.data_ptr()
    _op.call("flame_group_norm", device, x.data_ptr(), _op.ptr(weight), _op.ptr(bias), y.data_ptr(), _op.ptr(codes), _op.ptr(scales),
             at + size if stats is None else stats.data_ptr(), b, l, c, groups, eps, activation, _param_dtype(weight, bias), at, size)
    return y, stats, codes, scales


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation, codes_wanted):
        y, stats, codes, scales = _forward(x, weight, bias, groups, eps, activation, codes_wanted, True)
        ctx.groups, ctx.activation = groups, activation
        ctx.save_for_backward(x, weight, bias, stats)
        if not codes_wanted:
            return y
        ctx.mark_non_differentiable(codes, scales)
        return y, codes, scales

    @_op.first_order
    def backward(ctx, dy, *_):
        x, weight, bias, stats = (t if t is None else t.contiguous() for t in ctx.saved_tensors)      # hooks may give them other strides
        device, groups = x.device, ctx.groups
        b, l, c = _sizes(x)
        dy = dy.contiguous()
        dx = torch.empty_like(x)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        size = _workspace_bytes(device.index, b, l, c, groups, 1)
        ws = _op.workspace(x, size)
        _op.call("flame_group_norm_backward", device, x.data_ptr(), dy.data_ptr(), _op.ptr(weight), _op.ptr(bias), stats.data_ptr(),
                 dx.data_ptr(), _op.ptr(dw), _op.ptr(db), b, l, c, groups, ctx.activation, _param_dtype(weight, bias), ws.data_ptr(), size)
        return dx if ctx.needs_input_grad[0] else None, dw, db, None, None, None, None


def _param_dtype(weight, bias) -> int:
    t = weight if weight is not None else bias
    return 0 if t is None else _op.DTYPE[t.dtype]


def _check(what, x, groups, weight, bias, activation):
    _op.on_gpu(what, x, weight, bias)
    if x.dtype != torch.bfloat16 or x.dim() < 2 or not x.is_contiguous():
        raise InvalidInput(f"{what}: x must be a contiguous BF16 tensor [batch, ..., channels]")
    c = x.shape[-1]
    if not isinstance(groups, int) or groups <= 0 or c <= 0 or c % groups != 0:
        raise InvalidInput(f"{what}: {c} channels are not a multiple of {groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and not (t.dim() == 1 and t.shape[0] == c and t.is_contiguous() and t.dtype in _op.DTYPE):
            raise InvalidInput(f"{what}: {name} must be a contiguous BF16 or F32 vector of {c} elements")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise InvalidInput(f"{what}: weight and bias must have one type")
    if activation not in _ACTIVATIONS:
        raise InvalidInput(f"{what}: activation must be None, 'none' or 'silu'")


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """``act((x - mean) * rstd * weight + bias)`` with mean and variance of each sample's groups of channels."""
    _check("group_norm", x, groups, weight, bias, activation)
    if not _op.recorded(x, weight, bias):
        return _forward(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], False, False)[0]
    return _GroupNorm.apply(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], False)


def group_norm_fp8(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                   eps: float = 1e-5, activation: Optional[str] = None) -> Tuple[torch.Tensor, Fp8Blocks]:
    """``group_norm`` and the FP8 codes of its output (one scale for 128 channels of a position; channels % 128 == 0).

    The codes are those ``quantize_fp8(y, "rows")`` gives; ``fp8_linear(y, weight, codes=codes)`` reads them in place of ``y``."""
    _check("group_norm_fp8", x, groups, weight, bias, activation)
    if x.shape[-1] % 128 != 0 or x.data_ptr() % 16 != 0:
        raise InvalidInput("group_norm_fp8: channels must be a multiple of 128, and x must start on 16 bytes")
    if _op.recorded(x, weight, bias):
        y, codes, scales = _GroupNorm.apply(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], True)
    else:
        y, _, codes, scales = _forward(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], True, False)
    return y, Fp8Blocks(codes, scales, "rows")
