"""Matrix products of FP8 operands with one scale for each block of 128, and the linear layer made of them.

The weight path of this package expands FP8 bytes to BF16 before a product (``fused_inference``); here the tensor cores read the
codes as they are.  A block runs along the contraction: ``rows`` (1 x 128), ``columns`` (128 x 1) or ``tiles`` (128 x 128, a
weight, whose codes serve the product and its transpose).

    q = quantize_fp8(w, "tiles")              # once, for a frozen weight
    y = fp8_linear(x, q)                      # y = x w^T; gradients flow to x
    y = fp8_linear(x, w)                      # w a BF16 parameter: quantised in the call, gradients to both

Codes are OCP E4M3 (round to nearest even, saturating at 448).  Codes of the reference's encoder, the pool's FP8 default, are no
operands: there code 0x7F stands for 480.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _op
from ._op import need
from .errors import InvalidShape, Unsupported

BLOCK = 128
_BLOCKS = {"rows": 1, "columns": 2, "tiles": 3}     # FLAME_FP8_BLOCKS_*


def _blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _scales_shape(rows: int, cols: int, blocks: str) -> Tuple[int, int]:
    return (rows if blocks == "rows" else _blocks_of(rows), cols if blocks == "columns" else _blocks_of(cols))


@dataclass(frozen=True)
class Fp8Blocks:
    """An FP8 matrix: uint8 ``codes`` [rows, cols] whose rows start 16 bytes or a multiple of it apart, and fp32 ``scales``:
    [rows, ceil(cols/128)] for "rows", [ceil(rows/128), cols] for "columns", [ceil(rows/128), ceil(cols/128)] for "tiles"."""

    codes: torch.Tensor
    scales: torch.Tensor
    blocks: str

    def __post_init__(self):
        need(self.blocks in _BLOCKS, f"Fp8Blocks: blocks must be one of {', '.join(_BLOCKS)}")
        c, s = self.codes, self.scales
        _op.on_gpu("Fp8Blocks", c, s)
        need(c.dtype == torch.uint8 and c.dim() == 2 and s.dtype == torch.float32 and s.is_contiguous(),
             "Fp8Blocks: uint8 codes [rows, cols] and contiguous float32 scales")
        need(tuple(s.shape) == _scales_shape(c.shape[0], c.shape[1], self.blocks),
             f"Fp8Blocks: scales {tuple(s.shape)} for codes {tuple(c.shape)}, expected {_scales_shape(c.shape[0], c.shape[1], self.blocks)}", InvalidShape)
        if c.numel():
            need((c.stride(1) == 1 or c.shape[1] == 1) and c.data_ptr() % 16 == 0, "Fp8Blocks: codes must be row-major and start on 16 bytes")
            need(c.shape[0] == 1 or (c.stride(0) % 16 == 0 and c.stride(0) >= c.shape[1]), "Fp8Blocks: rows of codes must be a multiple of 16 bytes apart")

    @property
    def shape(self) -> Tuple[int, int]:
        return tuple(self.codes.shape)

    @property
    def stride(self) -> int:
        """Bytes from row to row.  A matrix of one row may be the start of longer memory: its stride is its own length."""
        c = self.codes
        return c.stride(0) if c.shape[0] > 1 and c.shape[1] else _padded(c.shape[1])

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """code * scale as a new BF16 or F32 matrix."""
        need(dtype in _op.DTYPE, "dequantize: BF16 or F32")
        rows, cols = self.shape
        out = torch.empty(rows, cols, dtype=dtype, device=self.codes.device)
        _op.call("flame_fp8_dequant_2d", out.device, self.codes.data_ptr(), self.stride, self.scales.data_ptr(), _BLOCKS[self.blocks],
                 out.data_ptr(), _op.DTYPE[dtype], rows, cols)
        return out


def _padded(cols: int) -> int:
    return max(16, (cols + 15) // 16 * 16)


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as a BF16 matrix with neighbouring columns, without a copy."""
    need(x.dtype == torch.bfloat16 and x.dim() >= 1, f"{what}: BF16 tensors")
    if x.dim() != 2:
        need(x.is_contiguous(), f"{what}: a tensor of other than two dimensions must be contiguous")
        x = x.view(_rows_of(x), x.shape[-1])
    need(x.numel() == 0 or ((x.stride(1) == 1 or x.shape[1] == 1) and (x.shape[0] == 1 or x.stride(0) >= x.shape[1])),
         f"{what}: the columns of a matrix must be neighbours, and its rows must not overlap")
    return x


def _rows_of(x: torch.Tensor) -> int:
    n = 1
    for s in x.shape[:-1]:
        n *= s
    return n


def _quantize(x, blocks: Optional[str], columns: bool):
    rows, cols = x.shape
    ld = _padded(cols)

    def make(kind):
        return (torch.empty(rows, ld, dtype=torch.uint8, device=x.device),
                torch.empty(_scales_shape(rows, cols, kind), dtype=torch.float32, device=x.device))

    c, s = make(blocks) if blocks else (None, None)
    cc, cs = make("columns") if columns else (None, None)
    stride = x.stride(0) if rows > 1 else cols
    _op.call("flame_fp8_quant_2d", x.device, x.data_ptr(), rows, cols, stride, _op.ptr(c), _op.ptr(s), _BLOCKS[blocks] if blocks else 0,
             _op.ptr(cc), _op.ptr(cs), ld)
    out = []
    if blocks:
        out.append(Fp8Blocks(c[:, :cols], s, blocks))
    if columns:
        out.append(Fp8Blocks(cc[:, :cols], cs, "columns"))
    return out


def quantize_fp8(x: torch.Tensor, blocks: str = "rows") -> Fp8Blocks:
    """FP8 codes of a BF16 matrix (or of the rows of a contiguous tensor's last dimension)."""
    _op.on_gpu("quantize_fp8", x)
    need(blocks in _BLOCKS, f"quantize_fp8: blocks must be one of {', '.join(_BLOCKS)}")
    x = _matrix(x, "quantize_fp8")
    return _quantize(x, None, True)[0] if blocks == "columns" else _quantize(x, blocks, False)[0]


def quantize_fp8_both(x: torch.Tensor) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """``quantize_fp8(x, "rows")`` and ``quantize_fp8(x, "columns")`` from one read of x: what backward needs of an output gradient."""
    _op.on_gpu("quantize_fp8_both", x)
    rows, columns = _quantize(_matrix(x, "quantize_fp8_both"), "rows", True)
    return rows, columns


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, *, transpose_b: bool = False, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of two FP8 matrices as a BF16 or F32 matrix, summed in fp32.  The blocks say which product it is:

    * a "rows" [M, K], b "rows" or "tiles" [N, K], ``transpose_b=True``:  a b^T
    * a "rows" [M, K], b "tiles" [K, N]:                                 a b
    * a "columns" [K, M], b "columns" [K, N]:                            a^T b
    """
    need(isinstance(a, Fp8Blocks) and isinstance(b, Fp8Blocks), "fp8_matmul: Fp8Blocks operands")
    need(dtype in _op.DTYPE, "fp8_matmul: the result is BF16 or F32")
    device = _op.on_gpu("fp8_matmul", a.codes, b.codes)
    kinds = (a.blocks, b.blocks, bool(transpose_b))
    if kinds in (("rows", "rows", True), ("rows", "tiles", True)):
        (m, k), (n, kb) = a.shape, b.shape
    elif kinds == ("rows", "tiles", False):
        (m, k), (kb, n) = a.shape, b.shape
    elif kinds == ("columns", "columns", False):
        (k, m), (kb, n) = a.shape, b.shape
    else:
        raise Unsupported(f"fp8_matmul: no product of {a.blocks} and {b.blocks}{' transposed' if transpose_b else ''}: "
                          "the blocks must run along the contraction")
    need(k == kb, f"fp8_matmul: shapes {a.shape} and {b.shape} do not fit", InvalidShape)
    c = torch.empty(m, n, dtype=dtype, device=device)
    _op.call("flame_fp8_product", device, a.codes.data_ptr(), a.stride, a.scales.data_ptr(), _BLOCKS[a.blocks], b.codes.data_ptr(), b.stride,
             b.scales.data_ptr(), _BLOCKS[b.blocks], int(bool(transpose_b)), c.data_ptr(), n, _op.DTYPE[dtype], m, n, k)
    return c


class _Linear(torch.autograd.Function):
    """y = x w^T.  Saved for backward: x where the weight is trained (BF16, so that a pool can offload it), and the weight's codes."""

    @staticmethod
    def forward(ctx, x, weight, x_codes, x_scales, w_codes, w_scales, w_blocks):
        m = _matrix(x, "fp8_linear")
        qx = Fp8Blocks(x_codes, x_scales, "rows") if x_codes is not None else _quantize(m, "rows", False)[0]
        qw = Fp8Blocks(w_codes, w_scales, w_blocks) if w_codes is not None else _quantize(_matrix(weight, "fp8_linear"), "tiles", False)[0]
        y = fp8_matmul(qx, qw, transpose_b=True)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None,
                              *((qw.codes, qw.scales) if ctx.needs_input_grad[0] else (None, None)))
        ctx.shapes = (x.shape, qw.shape)
        return y.view(*x.shape[:-1], qw.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_codes, w_scales = ctx.saved_tensors
        x_shape, (n, k) = ctx.shapes
        dy = dy.contiguous().view(_rows_of(dy), n)
        want_dx, want_dw = ctx.needs_input_grad[:2]
        q = _quantize(dy, "rows" if want_dx else None, want_dw)
        dx = fp8_matmul(q[0], Fp8Blocks(w_codes, w_scales, "tiles")).view(x_shape) if want_dx else None
        dw = fp8_matmul(q[-1], _quantize(_matrix(x, "fp8_linear"), None, True)[0]) if want_dw else None
        return dx, dw, None, None, None, None, None


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Blocks], *, codes: Optional[Fp8Blocks] = None) -> torch.Tensor:
    """``x @ weight.T`` with both operands in FP8: x BF16 [..., K], weight [N, K].

    ``weight`` as ``Fp8Blocks`` is frozen ("tiles", or "rows" where x needs no gradient); as a BF16 tensor it is quantised in the call and
    receives a gradient.  ``codes``: the "rows" codes of x where a producer has written them already (``group_norm_fp8``)."""
    frozen = isinstance(weight, Fp8Blocks)
    w = weight.codes if frozen else weight
    _op.on_gpu("fp8_linear", x, w, codes.codes if codes is not None else None)
    if not frozen:
        need(weight.dtype == torch.bfloat16, "fp8_linear: the weight is a BF16 matrix or Fp8Blocks")
    need(w.dim() == 2, "fp8_linear: the weight is a matrix [N, K]")
    need(x.dtype == torch.bfloat16 and x.dim() >= 1 and x.shape[-1] == w.shape[1],
         f"fp8_linear: x {tuple(x.shape)} and weight {tuple(w.shape)} do not fit", InvalidShape)
    if frozen:
        need(weight.blocks != "columns", "fp8_linear: the blocks of a weight are tiles or rows", Unsupported)
        need(weight.blocks == "tiles" or not (torch.is_grad_enabled() and x.requires_grad),
             "fp8_linear: a weight with rows of blocks has no input gradient; quantise it to tiles", Unsupported)
    if codes is not None:
        need(codes.blocks == "rows" and codes.shape == (_rows_of(x), x.shape[-1]), "fp8_linear: codes must be the rows of x", InvalidShape)
    return _Linear.apply(x, None if frozen else weight, codes.codes if codes is not None else None, codes.scales if codes is not None else None,
                         weight.codes if frozen else None, weight.scales if frozen else None, weight.blocks if frozen else None)
