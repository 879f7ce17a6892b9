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

import ctypes
import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib, _op
from .errors import CudaError, InvalidInput, InvalidShape, Unsupported

BLOCK = 128
_BLOCKS = {"rows": 1, "columns": 2, "tiles": 3}     # FLAME_FP8_BLOCKS_*


def _blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _scales_shape(rows: int, cols: int, blocks: str) -> Tuple[int, int]:
    return (rows if blocks == "rows" else _blocks_of(rows), cols if blocks == "columns" else _blocks_of(cols))


def _padded(cols: int) -> int:
    return max(16, (cols + 15) // 16 * 16)


class Fp8Blocks:
    """An FP8 matrix: uint8 ``codes`` [rows, cols] whose rows start 16 bytes or a multiple of it apart, and fp32 ``scales``:
    [rows, ceil(cols/128)] for "rows", [ceil(rows/128), cols] for "columns", [ceil(rows/128), ceil(cols/128)] for "tiles"."""

    __slots__ = ("codes", "scales", "blocks", "shape", "stride")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, blocks: str):
        if blocks not in _BLOCKS:
            raise InvalidInput(f"Fp8Blocks: blocks must be one of {', '.join(_BLOCKS)}")
        _op.on_gpu("Fp8Blocks", codes, scales)
        if codes.dtype != torch.uint8 or codes.dim() != 2 or scales.dtype != torch.float32 or not scales.is_contiguous():
            raise InvalidInput("Fp8Blocks: uint8 codes [rows, cols] and contiguous float32 scales")
        rows, cols = codes.shape
        want = _scales_shape(rows, cols, blocks)
        if scales.shape != want:
            raise InvalidShape(f"Fp8Blocks: scales {tuple(scales.shape)} for codes {(rows, cols)}, expected {want}")
        # a matrix of one row may be the start of longer memory: its stride is its own length
        stride = codes.stride(0) if rows > 1 and cols else _padded(cols)
        if rows and cols:
            if (codes.stride(1) != 1 and cols != 1) or codes.data_ptr() % 16 != 0:
                raise InvalidInput("Fp8Blocks: codes must be row-major and start on 16 bytes")
            if stride % 16 != 0 or stride < cols:
                raise InvalidInput("Fp8Blocks: rows of codes must be a multiple of 16 bytes apart")
        self.codes, self.scales, self.blocks, self.shape, self.stride = codes, scales, blocks, (rows, cols), stride

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """code * scale as a new BF16 or F32 matrix."""
        if dtype not in _op.DTYPE:
            raise InvalidInput("dequantize: BF16 or F32")
        rows, cols = self.shape
        out = torch.empty(rows, cols, dtype=dtype, device=self.codes.device)
        _op.call("flame_fp8_dequant_2d", out.device, self.codes.data_ptr(), self.stride, self.scales.data_ptr(), _BLOCKS[self.blocks],
                 out.data_ptr(), _op.DTYPE[dtype], rows, cols)
        return out


def _rows_of(shape) -> int:
    n = 1
    for s in shape[:-1]:
        n *= s
    return n


def _matrix(x: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(rows, columns, elements from row to row) of a BF16 tensor read as a matrix of its last dimension."""
    if x.dtype != torch.bfloat16 or x.dim() < 1:
        raise InvalidInput(f"{what}: BF16 tensors of one dimension at least")
    shape = x.shape
    cols = shape[-1]
    rows = shape[0] if len(shape) == 2 else _rows_of(shape)
    if x.is_contiguous():
        return rows, cols, cols
    if x.dim() != 2:
        raise InvalidInput(f"{what}: a tensor of other than two dimensions must be contiguous")
    if (x.stride(1) != 1 and cols != 1) or (rows != 1 and x.stride(0) < cols):
        raise InvalidInput(f"{what}: the columns of a matrix must be neighbours, and its rows must not overlap")
    return rows, cols, x.stride(0) if rows > 1 else cols


def _quantize(x, what, blocks: Optional[str], columns: bool):
    _op.on_gpu(what, x)
    rows, cols, stride = _matrix(x, what)
    ld = _padded(cols)

    def make(kind):
        return (torch.empty(rows, ld, dtype=torch.uint8, device=x.device),
                torch.empty(_scales_shape(rows, cols, kind), dtype=torch.float32, device=x.device))

    c, s = make(blocks) if blocks else (None, None)
    cc, cs = make("columns") if columns else (None, None)
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
    if blocks not in _BLOCKS:
        raise InvalidInput(f"quantize_fp8: blocks must be one of {', '.join(_BLOCKS)}")
    columns = blocks == "columns"
    return _quantize(x, "quantize_fp8", None if columns else blocks, columns)[0]


def quantize_fp8_both(x: torch.Tensor) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """``quantize_fp8(x, "rows")`` and ``quantize_fp8(x, "columns")`` from one read of x."""
    rows, columns = _quantize(x, "quantize_fp8_both", "rows", True)
    return rows, columns


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, *, transpose_b: bool = False, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of two FP8 matrices as a BF16 or F32 matrix, summed in fp32.  The blocks say which product it is:

    * a "rows" [M, K], b "rows" or "tiles" [N, K], ``transpose_b=True``:  a b^T
    * a "rows" [M, K], b "tiles" [K, N]:                                 a b
    * a "columns" [K, M], b "columns" [K, N]:                            a^T b
    """
    if not (isinstance(a, Fp8Blocks) and isinstance(b, Fp8Blocks)):
        raise InvalidInput("fp8_matmul: Fp8Blocks operands")
    if dtype not in _op.DTYPE:
        raise InvalidInput("fp8_matmul: the result is BF16 or F32")
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
    if k != kb:
        raise InvalidShape(f"fp8_matmul: shapes {a.shape} and {b.shape} do not fit")
    c = torch.empty(m, n, dtype=dtype, device=device)
    _op.call("flame_fp8_product", device, a.codes.data_ptr(), a.stride, a.scales.data_ptr(), _BLOCKS[a.blocks], b.codes.data_ptr(), b.stride,
             b.scales.data_ptr(), _BLOCKS[b.blocks], int(bool(transpose_b)), c.data_ptr(), n, _op.DTYPE[dtype], m, n, k)
    return c


_seen_faults: dict = {}


def check_faults(device: Optional[torch.device] = None) -> None:
    """Raises ``CudaError`` where a wait inside a product's kernel has given up since the last check: such a product wrote NaN where its
    result is not known.  Waits for the device (the current one by default), so it belongs where a program waits for it anyway."""
    index = torch.device(device).index if device is not None else None
    if index is None:
        index = torch.cuda.current_device()
    count = ctypes.c_uint(0)
    with torch.cuda.device(index):
        rc = _op.function("flame_fp8_product_faults")(ctypes.byref(count))
    if rc:
        raise CudaError(f"flame_fp8_product_faults failed ({rc}): {_lib.last_error()}")
    new = count.value - _seen_faults.get(index, 0)
    _seen_faults[index] = count.value
    if new:
        raise CudaError(f"FP8 product: {new} warps on GPU {index} gave up a wait; the products concerned hold NaN")


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m: int, n: int, k: int, flags: int) -> int:
    return max(_op.function("flame_fp8_linear_workspace_bytes")(m, n, k, flags), 16)


def _weight_args(weight, frozen: Optional[Fp8Blocks]):
    """(N, the library's arguments for the weight): BF16, or codes that somebody keeps."""
    if frozen is not None:
        return frozen.shape[0], (None, 0, frozen.codes.data_ptr(), frozen.stride, frozen.scales.data_ptr())
    n, _, stride = _matrix(weight, "fp8_linear")
    return n, (weight.data_ptr(), stride, None, 0, None)


def _forward(x, codes: Optional[Fp8Blocks], weight, frozen: Optional[Fp8Blocks]) -> torch.Tensor:
    m, k, x_stride = _matrix(x, "fp8_linear")
    n, w_args = _weight_args(weight, frozen)
    y = x.new_empty(x.shape[:-1] + (n,))
    size = _workspace_bytes(m, n, k, 0 if frozen is not None else 2)      # FLAME_FP8_LINEAR_BF16_WEIGHT
    ws = _op.workspace(x, size)
    given = (None, 0, None) if codes is None else (codes.codes.data_ptr(), codes.stride, codes.scales.data_ptr())
    _op.call("flame_fp8_linear", x.device, x.data_ptr(), x_stride, *given, *w_args, 3 if frozen is None else _BLOCKS[frozen.blocks], y.data_ptr(), m, n, k,
             ws.data_ptr(), size)
    return y


def _rows_again(t: torch.Tensor) -> torch.Tensor:
    """A saved BF16 tensor as ``_matrix`` reads it: hooks may give it back with strides of their own."""
    cols = t.shape[-1]
    if t.is_contiguous() or (t.dim() == 2 and (t.stride(1) == 1 or cols == 1) and (t.shape[0] == 1 or t.stride(0) >= cols)):
        return t
    return t.contiguous()


def _codes_again(codes: torch.Tensor) -> torch.Tensor:
    """Saved codes as ``Fp8Blocks`` takes them: hooks that copy leave out the padding of the rows."""
    rows, cols = codes.shape
    if rows == 0 or cols == 0:
        return codes
    if (codes.stride(1) == 1 or cols == 1) and codes.data_ptr() % 16 == 0 and (rows == 1 or (codes.stride(0) % 16 == 0 and codes.stride(0) >= cols)):
        return codes
    padded = codes.new_empty(rows, _padded(cols))[:, :cols]
    return padded.copy_(codes)


class _Linear(torch.autograd.Function):
    """y = x w^T.  Saved for backward: x where the weight is trained (BF16, so that a pool can offload it) and the weight itself.  Its codes
    are made again: keeping them would hold half as much memory again as the weights do, for a few per cent of a step's time."""

    @staticmethod
    def forward(ctx, x, weight, codes, frozen):
        y = _forward(x, codes, weight, frozen)
        want_dx, want_dw = ctx.needs_input_grad[:2]
        kept = (frozen.codes, frozen.scales) if frozen is not None else (weight, None)
        ctx.save_for_backward(x if want_dw else None, *(kept if want_dx else (None, None)))
        ctx.frozen = frozen is not None
        ctx.x_shape, ctx.n = x.shape, y.shape[-1]
        return y

    @_op.first_order
    def backward(ctx, dy):
        x, w, w_scales = ctx.saved_tensors
        want_dx, want_dw = ctx.needs_input_grad[:2]
        shape, n = ctx.x_shape, ctx.n
        device = dy.device
        dy = dy.contiguous()
        m, k = _rows_of(shape), shape[-1]
        dx = dy.new_empty(shape) if want_dx else None
        dw = dy.new_empty(n, k) if want_dw else None
        w_args = (None, 0, None, 0, None)
        if want_dw:
            x = _rows_again(x)
        if want_dx:
            w, w_scales = (_codes_again(w), w_scales.contiguous()) if ctx.frozen else (_rows_again(w), None)
            w_args = _weight_args(w, Fp8Blocks(w, w_scales, "tiles") if ctx.frozen else None)[1]
        size = _workspace_bytes(m, n, k, 1 if ctx.frozen else 3)
        ws = _op.workspace(dy, size)
        _op.call("flame_fp8_linear_backward", device, dy.data_ptr(), n, _op.ptr(x), _matrix(x, "fp8_linear")[2] if want_dw else 0, *w_args,
                 _op.ptr(dx), _op.ptr(dw), m, n, k, ws.data_ptr(), size)
        return dx, dw, None, None


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Blocks], *, codes: Optional[Fp8Blocks] = None) -> torch.Tensor:
    """``x @ weight.T`` with both operands in FP8: x BF16 [..., K], weight [N, K].

    ``weight`` as ``Fp8Blocks`` is frozen ("tiles", or "rows" where x needs no gradient); as a BF16 tensor it is quantised in the call and
    receives a gradient.  ``codes``: the "rows" codes of x where a producer has written them already (``group_norm_fp8``)."""
    frozen = weight if isinstance(weight, Fp8Blocks) else None
    if frozen is None and not isinstance(weight, torch.Tensor):
        raise InvalidInput(f"fp8_linear: expected a tensor or Fp8Blocks as weight, got {type(weight).__name__}")
    if codes is not None and not isinstance(codes, Fp8Blocks):
        raise InvalidInput(f"fp8_linear: codes are Fp8Blocks, got {type(codes).__name__}")
    _op.on_gpu("fp8_linear", x, weight if frozen is None else frozen.codes, codes.codes if codes is not None else None)
    if frozen is None and (weight.dtype != torch.bfloat16 or weight.dim() != 2):
        raise InvalidInput("fp8_linear: the weight is a BF16 matrix [N, K] or Fp8Blocks")
    w_shape = weight.shape
    if x.dtype != torch.bfloat16 or x.dim() < 1 or x.shape[-1] != w_shape[1]:
        raise InvalidShape(f"fp8_linear: x {x.dtype} {tuple(x.shape)} and weight {tuple(w_shape)} do not fit")
    if codes is not None and (codes.blocks != "rows" or codes.shape != (_rows_of(x.shape), x.shape[-1])):
        raise InvalidShape("fp8_linear: codes must be the rows of x")
    record = _op.recorded(x, None if frozen is not None else weight)
    if frozen is not None and frozen.blocks != "tiles":
        if frozen.blocks == "columns":
            raise Unsupported("fp8_linear: the blocks of a weight are tiles or rows")
        if record:
            raise Unsupported("fp8_linear: a weight with rows of blocks has no input gradient; quantise it to tiles")
    if not record:
        return _forward(x, codes, None if frozen is not None else weight, frozen)
    return _Linear.apply(x, None if frozen is not None else weight, codes, frozen)
