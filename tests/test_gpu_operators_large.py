"""Tensors of more than 2^31 elements: what lies behind that border equals what a call on that part alone gives."""
import numpy as np
import pytest
import torch

from flame_b200.dropout import dropout
from flame_b200.fp8_product import Fp8Blocks, fp8_matmul, quantize_fp8
from flame_b200.group_norm import group_norm

pytestmark = pytest.mark.gpu

BORDER = 1 << 31


@pytest.fixture(autouse=True)
def memory(cuda_device):
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    yield
    torch.cuda.empty_cache()


def keep(first, count, p, seed, offset):
    """The generator's definition for elements first .. first + count; first is a multiple of 8."""
    low, blk = np.uint64(0xFFFFFFFF), np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)

    def halves(top):
        c = [blk & low, blk >> np.uint64(32) | np.uint64(top), np.full_like(blk, offset), np.zeros_like(blk)]
        k = [seed, 0]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return np.stack(c, axis=1).astype("<u4").view("<u2").reshape(-1)[:count].astype(np.uint64)

    return (halves(0) << np.uint64(16) | halves(1 << 31)) >= round(p * 2 ** 32)


@pytest.mark.parametrize("start", [0, 1])      # whole groups of eight, and element by element
def test_dropout(cuda_device, start):
    n = BORDER + (1 << 20) + 5
    x = torch.ones(n + start, dtype=torch.bfloat16, device=cuda_device)[start:]
    y = dropout(x, 0.3, seed=7, offset=2)
    for first in (0, BORDER - 4096, n // 8 * 8 - 8192):
        count = min(n - first, 8197)
        assert np.array_equal((y[first:first + count] != 0).cpu().numpy(), keep(first, count, 0.3, 7, 2))


def test_group_norm(cuda_device):
    b, l, c = 2, (1 << 20) + 3, 1088
    assert b * l * c > BORDER
    x = torch.empty(b, l, c, dtype=torch.bfloat16, device=cuda_device).normal_().requires_grad_(True)
    w = (1 + 0.3 * torch.randn(c, device=cuda_device)).requires_grad_(True)
    y = group_norm(x, 32, w, activation="silu")
    dy = torch.empty_like(x).normal_()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    parts = []
    for i in range(b):
        alone = x.detach()[i:i + 1].requires_grad_(True)
        z = group_norm(alone, 32, w, activation="silu")
        dz, part = torch.autograd.grad(z, (alone, w), dy[i:i + 1])
        parts.append(part)
        # other chunks: the statistics differ in their last bits, an element by one step of BF16, and near zero by 2^-18 of what is added up
        for got, want in ((y.detach()[i], z.detach()[0]), (dx[i], dz[0])):
            for rows in (slice(0, 1000), slice(l // 2, l // 2 + 1000), slice(l - 1000, l)):
                assert torch.allclose(got[rows].float(), want[rows].float(), rtol=2.0 ** -7, atol=2.0 ** -14)
    # sums over 2^21 positions in two orders: chains of some 2,000 additions, each off by 2^-24 of a partial sum of the size of the root of
    # their number at most, some 2^-13 of it, and the parts' sums besides
    want = parts[0].double() + parts[1].double()
    assert bool(((dw.double() - want).abs() <= 2.0 ** -10 * (b * l) ** 0.5).all())


def test_quantiser_and_dequantiser(cuda_device):
    rows, cols = (1 << 20) + 1, 2056
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda_device).normal_()
    at = rows // 128 * 128 - 256
    for blocks in ("rows", "columns", "tiles"):
        q, tail = quantize_fp8(x, blocks), quantize_fp8(x[at:], blocks)
        assert torch.equal(q.codes[at:], tail.codes) and torch.equal(q.scales[at if blocks == "rows" else at // 128:], tail.scales)
        assert torch.equal(q.dequantize(torch.bfloat16)[at:], tail.dequantize(torch.bfloat16))


@pytest.mark.parametrize("k", [16, 300])
def test_product(cuda_device, k):
    m = n = 46400
    assert m * n > BORDER
    g = torch.Generator(device=cuda_device).manual_seed(k)

    def integers(shape, blocks):
        codes = torch.zeros(shape[0], (shape[1] + 15) // 16 * 16, dtype=torch.uint8, device=cuda_device)
        codes[:, :shape[1]] = torch.randint(-8, 9, shape, device=cuda_device, generator=g).float().to(torch.float8_e4m3fn).view(torch.uint8)
        scales = torch.ones(shape[0] if blocks == "rows" else -(-shape[0] // 128), -(-shape[1] // 128), device=cuda_device)
        return Fp8Blocks(codes[:, :shape[1]], scales, blocks)

    a, b = integers((m, k), "rows"), integers((n, k), "tiles")
    c = fp8_matmul(a, b, transpose_b=True)
    x, y = (t.codes.contiguous().view(torch.float8_e4m3fn).double() for t in (a, b))
    for rows in (slice(0, 300), slice(m - 300, m)):
        for cols in (slice(0, 300), slice(n - 300, n)):
            assert torch.equal(c[rows, cols], (x[rows] @ y[cols].T).to(torch.bfloat16))
