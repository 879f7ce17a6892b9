"""Dropout against the generator's definition in whole numbers."""
import numpy as np
import pytest
import torch

from flame_b200 import InvalidInput
from flame_b200 import checkpoint as ckpt
from flame_b200.dropout import dropout

pytestmark = pytest.mark.gpu


def philox(c, key):
    c, (k0, k1) = list(c), key
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k1, a & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def bits(i, seed, offset):
    """u(i) in Python's integers."""
    g, j = divmod(i, 8)
    key = (seed & 0xFFFFFFFF, seed >> 32)
    half = lambda top: philox([g & 0xFFFFFFFF, g >> 32 | top, offset & 0xFFFFFFFF, offset >> 32], key)[j // 2] >> (16 * (j & 1)) & 0xFFFF  # noqa: E731
    return half(0) << 16 | half(1 << 31)


def kept(n, p, seed, offset):
    return torch.tensor([bits(i, seed, offset) >= round(p * 2 ** 32) for i in range(n)])


def test_known_numbers_of_the_generator():
    """Two of the vectors published with the generator (the counter and key all zeros, all ones)."""
    assert philox([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert philox([f] * 4, (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,p,seed,offset", [(1, 0.5, 0, 0), (7, 0.1, 1, 2), (8, 0.3, 5, 0), (1000, 0.1, 2 ** 63 + 11, 2 ** 64 - 1), (4099, 0.9, 77, 2 ** 33),
                                             (513, 0.0, 3, 1), (513, 1.0, 3, 1), (2000, 1e-3, 9, 9)])
def test_values_and_gradient(cuda_device, dtype, n, p, seed, offset):
    g = torch.Generator(device=cuda_device).manual_seed(n)
    x, dy, r = (torch.randn(n, device=cuda_device, generator=g).to(dtype) for _ in range(3))
    keep = kept(n, p, seed, offset).to(cuda_device)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32, device=cuda_device)
    zero = torch.zeros((), device=cuda_device)
    want = torch.where(keep, x.float() * scale, zero)
    x.requires_grad_(True)
    y = dropout(x, p, seed=seed, offset=offset)
    assert torch.equal(y, want.to(dtype))                      # one product and one rounding: the same bits
    y.backward(dy)
    assert torch.equal(x.grad, torch.where(keep, dy.float() * scale, zero).to(dtype))
    # the map is linear: the difference in a direction v is the gradient's product with it, to the rounding of either
    r.requires_grad_(True)
    z = dropout(x, p, seed=seed, offset=offset, residual=r)
    assert torch.equal(z, (r.float() + want).to(dtype))
    x.grad = None
    z.backward(dy)
    assert torch.equal(x.grad, torch.where(keep, dy.float() * scale, zero).to(dtype)) and torch.equal(r.grad, dy)
    seed_tensor = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed], device=cuda_device)
    assert torch.equal(dropout(x, p, seed=seed_tensor, offset=offset), y)


def test_ties_of_the_upper_half_are_decided_by_the_lower(cuda_device):
    """p just above t/65536: elements whose upper 16 bits equal t depend on the lower 16.  The seed is one for which several of the
    first 2^17 elements do."""
    n, seed, offset, t = 1 << 17, 12, 3, 30000
    blk = np.arange(n // 8, dtype=np.uint64)

    def halves(top):
        low = np.uint64(0xFFFFFFFF)
        c = [blk & low, blk >> np.uint64(32) | np.uint64(top), np.full_like(blk, offset), np.zeros_like(blk)]
        k = [seed, 0]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return np.stack(c, axis=1).astype("<u4").view("<u2").reshape(-1).astype(np.uint64)

    u = halves(0) << np.uint64(16) | halves(1 << 31)
    ties = np.nonzero(u >> np.uint64(16) == t)[0]
    assert len(ties) >= 1 and all(int(u[i]) == bits(int(i), seed, offset) for i in ties)
    for i in ties:
        for threshold in (int(u[i]), int(u[i]) + 1):
            y = dropout(torch.ones(n, device=cuda_device), threshold / 2 ** 32, seed=seed, offset=offset)
            assert np.array_equal((y != 0).cpu().numpy(), u >= threshold)


def test_dropped_values_leave_nothing_and_the_rate_is_right(cuda_device):
    n, p = 1 << 20, 0.3
    x = torch.full((n,), float("inf"), device=cuda_device)
    x[::2] = float("nan")
    y = dropout(x, p, seed=4)
    keep = dropout(torch.ones(n, device=cuda_device), p, seed=4) != 0
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())
    # a binomial count of n trials: five standard deviations
    assert abs(float(keep.float().mean()) - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    other = dropout(torch.ones(n, device=cuda_device), p, seed=4, offset=1) != 0
    both = float((keep & other).float().mean())
    assert abs(both - (1 - p) ** 2) < 5 * (0.25 / n) ** 0.5      # masks of two offsets are independent


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unaligned_tensors_and_what_lies_behind(cuda_device, dtype):
    for n in (1, 9, 1001):
        base = torch.randn(n + 3, device=cuda_device).to(dtype)
        x = base[1:1 + n]
        assert torch.equal(dropout(x, 0.4, seed=9, offset=5), dropout(x.clone(), 0.4, seed=9, offset=5))
        r = base[2:2 + n]
        assert torch.equal(dropout(x.clone(), 0.4, seed=9, residual=r), dropout(x.clone(), 0.4, seed=9, residual=r.clone()))
        from flame_b200 import _lib
        out = torch.full((n + 2,), 7.0, dtype=dtype, device=cuda_device)
        x = x.clone()
        assert _lib.lib().flame_dropout(x.data_ptr(), None, out.data_ptr(), n, 0 if dtype == torch.bfloat16 else 1, 0.4, 9, None, 5, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[:n], dropout(x, 0.4, seed=9, offset=5)) and bool((out[n:] == 7).all())


def test_recomputation_draws_the_same_mask(cuda_device):
    """Under ``checkpoint`` the forward pass runs twice; nothing about the generator has to be saved between the two."""
    x = torch.randn(64, 256, device=cuda_device, dtype=torch.bfloat16)

    def f(t):
        return dropout(torch.sin(dropout(t, 0.2, seed=21, offset=0)), 0.2, seed=21, offset=1, residual=t)

    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ya, yb = f(a), ckpt.checkpoint([b], f)
    ya.sum().backward()
    yb.sum().backward()
    assert torch.equal(ya, yb) and torch.equal(a.grad, b.grad)


def test_replayed_graph_reads_the_next_seed(cuda_device):
    x = torch.randn(3000, device=cuda_device, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    seed = torch.tensor([5], device=cuda_device)

    def step(s):
        a = x.detach().requires_grad_(True)
        y = dropout(a, 0.25, seed=s, offset=2)
        return y.detach(), torch.autograd.grad(y, a, dy)[0]

    step(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(seed)
    for value in (5, 6, 700):
        seed.fill_(value)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, step(value)))
    a = x.clone().requires_grad_(True)
    y = dropout(a, 0.25, seed=seed, offset=2)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_side_stream_and_empty(cuda_device):
    x = torch.randn(1 << 16, device=cuda_device, dtype=torch.bfloat16)
    want = dropout(x, 0.5, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = dropout(x, 0.5, seed=1)
    side.synchronize()
    assert torch.equal(y, want)
    e = torch.empty(0, 8, device=cuda_device, requires_grad=True)
    dropout(e, 0.5, seed=1).sum().backward()
    assert e.grad.shape == (0, 8)


def test_refusals(cuda_device):
    x = torch.randn(8, 8, device=cuda_device)
    for kwargs, text in (({"p": 1.5}, "p must be"), ({"p": float("nan")}, "p must be"), ({"seed": -1}, "seed"), ({"seed": 2 ** 64}, "seed"), ({"offset": -1}, "offset"),
                         ({"seed": torch.tensor([1])}, "seed tensor"), ({"residual": x[:4]}, "residual"), ({"residual": x.bfloat16()}, "residual")):
        with pytest.raises(InvalidInput, match=text):
            dropout(**{"x": x, "p": 0.5, "seed": 1, **kwargs})
    with pytest.raises(InvalidInput, match="contiguous"):
        dropout(x.t(), 0.5, seed=1)
    with pytest.raises(InvalidInput, match="BF16 or F32"):
        dropout(x.half(), 0.5, seed=1)
    with pytest.raises(InvalidInput, match="on the GPU"):
        dropout(x.cpu(), 0.5, seed=1)
