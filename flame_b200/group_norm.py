"""Group norm with an activation on channels-last tensors, beside the RMSNorm producer.

``x`` is ``[batch, positions..., channels]``, BF16 and contiguous (a ``[B, C, H, W]`` tensor in channels-last memory is
``x.permute(0, 2, 3, 1)``).  The activation is part of both passes: backward needs ``x`` and two floats for each sample and group,
so a block saves one tensor for the norm and its activation, and a pool can offload it.
``group_norm_fp8`` also writes the FP8 codes of its output, the left operand of ``fp8_product.fp8_linear``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, _op
from ._op import need
from .fp8_product import Fp8Blocks

_ACTIVATIONS = {None: 0, "none": 0, "silu": 1}     # FLAME_ACTIVATION_*


def _workspace(x, b, l, c, groups, backward):
    with torch.cuda.device(x.device):
        n = _lib.lib().flame_group_norm_workspace_bytes(b, l, c, groups, backward)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)


def _sizes(x):
    b, c = x.shape[0], x.shape[-1]
    l = 1
    for n in x.shape[1:-1]:
        l *= n
    return b, l, c


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation, codes_wanted):
        b, l, c = _sizes(x)
        y = torch.empty_like(x)
        stats = torch.empty(b, groups, 2, dtype=torch.float32, device=x.device)
        codes = scales = None
        if codes_wanted:
            codes = torch.empty(b * l, c, dtype=torch.uint8, device=x.device)
            scales = torch.empty(b * l, c // 128, dtype=torch.float32, device=x.device)
        params = _param_dtype(weight, bias)
        ws = _workspace(x, b, l, c, groups, 0)
        _op.call("flame_group_norm", x.device, x.data_ptr(), _op.ptr(weight), _op.ptr(bias), y.data_ptr(), _op.ptr(codes), _op.ptr(scales),
                 stats.data_ptr(), b, l, c, groups, eps, activation, params, ws.data_ptr(), ws.numel())
        ctx.groups, ctx.activation = groups, activation
        ctx.save_for_backward(x, weight, bias, stats)
        if not codes_wanted:
            return y
        ctx.mark_non_differentiable(codes, scales)
        return y, codes, scales

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *_):
        x, weight, bias, stats = ctx.saved_tensors
        b, l, c = _sizes(x)
        dy = dy.contiguous()
        dx = torch.empty_like(x)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        ws = _workspace(x, b, l, c, ctx.groups, 1)
        _op.call("flame_group_norm_backward", x.device, x.data_ptr(), dy.data_ptr(), _op.ptr(weight), _op.ptr(bias), stats.data_ptr(),
                 dx.data_ptr(), _op.ptr(dw), _op.ptr(db), b, l, c, ctx.groups, ctx.activation, _param_dtype(weight, bias),
                 ws.data_ptr(), ws.numel())
        return dx if ctx.needs_input_grad[0] else None, dw, db, None, None, None, None


def _param_dtype(weight, bias) -> int:
    t = weight if weight is not None else bias
    return 0 if t is None else _op.DTYPE[t.dtype]


def _check(what, x, groups, weight, bias, activation):
    _op.on_gpu(what, x, weight, bias)
    need(x.dtype == torch.bfloat16 and x.dim() >= 2 and x.is_contiguous(), f"{what}: x must be a contiguous BF16 tensor [batch, ..., channels]")
    c = x.shape[-1]
    need(isinstance(groups, int) and groups > 0 and c > 0 and c % groups == 0, f"{what}: {c} channels are not a multiple of {groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            need(t.shape == (c,) and t.is_contiguous() and t.dtype in _op.DTYPE, f"{what}: {name} must be a contiguous BF16 or F32 vector of {c} elements")
    need(weight is None or bias is None or weight.dtype == bias.dtype, f"{what}: weight and bias must have one type")
    need(activation in _ACTIVATIONS, f"{what}: activation must be None, 'none' or 'silu'")


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """``act((x - mean) * rstd * weight + bias)`` with mean and variance of each sample's groups of channels."""
    _check("group_norm", x, groups, weight, bias, activation)
    return _GroupNorm.apply(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], False)


def group_norm_fp8(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                   eps: float = 1e-5, activation: Optional[str] = None) -> Tuple[torch.Tensor, Fp8Blocks]:
    """``group_norm`` and the FP8 codes of its output (one scale for 128 channels of a position; channels % 128 == 0).

    The codes are those ``quantize_fp8(y, "rows")`` gives; ``fp8_linear(y, weight, codes=codes)`` reads them in place of ``y``."""
    _check("group_norm_fp8", x, groups, weight, bias, activation)
    need(x.shape[-1] % 128 == 0, "group_norm_fp8: channels must be a multiple of 128")
    need(x.data_ptr() % 16 == 0, "group_norm_fp8: x must start on 16 bytes")
    y, codes, scales = _GroupNorm.apply(x, weight, bias, groups, float(eps), _ACTIVATIONS[activation], True)
    return y, Fp8Blocks(codes, scales, "rows")
