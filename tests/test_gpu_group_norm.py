"""Channels-last group norm with an activation, forward and backward, against 64-bit arithmetic."""
import pytest
import torch

from flame_b200 import ActivationOffloadPool, InvalidInput, OffloadCompression, _lib
from flame_b200 import checkpoint as ckpt
from flame_b200.fp8_product import fp8_linear, quantize_fp8
from flame_b200.group_norm import group_norm, group_norm_fp8

pytestmark = pytest.mark.gpu

# (batch, positions, channels, groups): vectors of 8, 2 and 1 channels; groups inside, across and of several vectors; one group, one
# channel a group; more channels than a thread block's width; one position
SHAPES = [(2, 64, 64, 8), (1, 1, 32, 4), (3, 100, 320, 32), (2, 33, 90, 6), (1, 257, 15, 3), (2, 50, 2560, 32), (1, 9, 4104, 9), (2, 7, 258, 1),
          (1, 40, 48, 48), (1, 5000, 128, 32), (4, 17, 8, 1), (2, 3, 771, 257), (1, 2, 1, 1)]


def reference(x, groups, weight, bias, eps, silu, dy):
    """Output and gradients in 64 bits from the formulas."""
    b, c = x.shape[0], x.shape[-1]
    x = x.double().reshape(b, -1, groups, c // groups)
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1 / ((x - mean).square().mean((1, 3), keepdim=True) + eps).sqrt()
    xhat = ((x - mean) * rstd).reshape(b, -1, c)
    w = weight.double() if weight is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    t = bias.double() if bias is not None else torch.zeros(c, dtype=torch.float64, device=x.device)
    h = xhat * w + t
    s = torch.sigmoid(h)
    y = h * s if silu else h
    dy = dy.double().reshape(b, -1, c)
    dh = dy * (s * (1 + h * (1 - s))) if silu else dy
    u = (dh * w).reshape(b, -1, groups, c // groups)
    xg = xhat.reshape(u.shape)
    dx = rstd * (u - u.mean((1, 3), keepdim=True) - xg * (u * xg).mean((1, 3), keepdim=True))
    # magnitudes that the roundings are relative to
    size_h = ((x.abs() + mean.abs()) * rstd).reshape(b, -1, c) * w.abs() + t.abs()
    size_u = (dy.abs() * 1.1 * (w.abs() + 1) * (1 + size_h)).reshape(u.shape)
    size_dx = rstd * (size_u + size_u.mean((1, 3), keepdim=True) * (1 + xg.abs()))
    return dict(y=y, dx=dx.reshape(b, -1, c), dw=(dh * xhat).sum((0, 1)), db=dh.sum((0, 1)), size_h=size_h,
                size_dx=size_dx.reshape(b, -1, c), size_dw=(1.1 * dy.abs() * (1 + size_h) * (1 + xhat.abs())).sum((0, 1)), size_db=(1.1 * dy.abs() * (1 + size_h)).sum((0, 1)))


def inputs(shape, device, params, offset=0.5):
    b, l, c, g = shape
    gen = torch.Generator(device=device).manual_seed(b + 3 * l + 7 * c + g)
    n = lambda *s: torch.randn(*s, device=device, generator=gen)  # noqa: E731
    x = (n(b, l, c) * (0.5 + torch.rand(c, device=device, generator=gen)) + offset * n(c)).to(torch.bfloat16)
    return x, (1 + 0.3 * n(c)).to(params), (0.3 * n(c)).to(params), n(b, l, c).to(torch.bfloat16)


# An element of the output takes some ten binary32 roundings, each 2^-24 of the magnitudes that enter it; the mean and the
# variance are sums over chains of at most a few hundred additions and the exponential is good to 2^-21: 2^-15 of the
# magnitudes bounds them together.  Then one rounding to BF16, 2^-8 of the value.
FP32, BF16 = 2.0 ** -15, 2.0 ** -8


@pytest.mark.parametrize("activation", ["silu", None])
@pytest.mark.parametrize("params", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_gradients(cuda_device, shape, params, activation):
    x, w, b, dy = inputs(shape, cuda_device, params or torch.float32)
    if params is None:
        w = b = None
    x.requires_grad_(True)
    leaves = [t.requires_grad_(True) for t in (w, b) if t is not None]
    y = group_norm(x, shape[3], w, b, eps=1e-5, activation=activation)
    y.backward(dy)
    r = reference(x.detach(), shape[3], w, b, 1e-5, activation == "silu", dy)
    assert bool(((y.detach().double() - r["y"]).abs() <= BF16 * r["y"].abs() + FP32 * r["size_h"]).all())
    assert bool(((x.grad.double() - r["dx"]).abs() <= BF16 * r["dx"].abs() + FP32 * r["size_dx"]).all())
    if leaves:
        last = BF16 if params == torch.bfloat16 else 0.0
        for got, name in ((w.grad, "dw"), (b.grad, "db")):
            assert got.dtype == params
            assert bool(((got.double() - r[name]).abs() <= last * r[name].abs() + FP32 * r["size_" + name]).all()), name


@pytest.mark.parametrize("activation", ["silu", None])
def test_gradients_against_differences(cuda_device, activation):
    """Central differences of the formula in 64 bits along random directions; step 2^-13, whose cubic term is under 2^-20 here."""
    shape = (2, 37, 48, 6)
    x, w, b, dy = inputs(shape, cuda_device, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(group_norm(*[leaves[0], 6, leaves[1], leaves[2]], activation=activation), leaves, dy)

    def loss(x, w, b):
        return float((reference(x, 6, w, b, 1e-5, activation == "silu", dy)["y"] * dy.double().view(2, -1, 48)).sum())

    gen = torch.Generator(device=cuda_device).manual_seed(1)
    for k, g in enumerate(grads):
        v = torch.randn(g.shape, device=cuda_device, generator=gen, dtype=torch.float64)
        h = 2.0 ** -13
        args = [t.detach().double() for t in leaves]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * v, args[k] - h * v
        slope = (loss(*up) - loss(*down)) / (2 * h)
        size = float((g.double().abs() * v.abs()).sum())
        assert abs(slope - float((g.double() * v).sum())) <= (BF16 if k == 0 else 2.0 ** -14) * size + 2.0 ** -14 * size


def test_mean_far_from_zero(cuda_device):
    """Values near 200 with steps of 1 and 2 (BF16 keeps 8 bits): sums of squares about zero would lose the variance."""
    x = (200 + torch.randint(-3, 4, (2, 4096, 64), device=cuda_device).float()).to(torch.bfloat16)
    y = group_norm(x, 8)
    r = reference(x, 8, None, None, 1e-5, False, torch.zeros_like(x))
    assert bool(((y.double() - r["y"]).abs() <= BF16 * r["y"].abs() + 2.0 ** -16).all())
    same = torch.full((1, 300, 32), 3.0, device=cuda_device, dtype=torch.bfloat16)      # no spread at all
    assert bool((group_norm(same, 4) == 0).all())


@pytest.mark.parametrize("positions", [1, 50, 4096, 200000])
def test_one_element_far_from_the_others(cuda_device, positions):
    """The first element of a group, a position's only large value: a sum of squares about it would lose the others.  A chunk has at most
    some thousand elements a group here, which err by n * 2^-24 of the outlier's square together: 2^-13 of the variance, half of that of
    the output."""
    x = torch.randn(1, positions, 32, device=cuda_device).to(torch.bfloat16)
    x[0, 0, 8] = 10000.0
    y = group_norm(x, 4)
    r = reference(x, 4, None, None, 1e-5, False, torch.zeros_like(x))
    assert bool(((y.double() - r["y"]).abs() <= (BF16 + 2.0 ** -14) * r["y"].abs() + FP32 * (1 + r["y"].abs())).all())


def test_nonfinite_values_stay_in_their_group(cuda_device):
    x, w, b, _ = inputs((2, 50, 64, 8), cuda_device, torch.float32)
    clean = group_norm(x, 8, w, b, activation="silu")
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[1, 20, 19] = bad                          # sample 1, channels 16..23
        y = group_norm(z, 8, w, b, activation="silu")
        assert bool(torch.isnan(y[1, :, 16:24]).all())
        y[1, :, 16:24] = clean[1, :, 16:24]
        assert torch.equal(y, clean)


def test_large_gate_values_do_not_overflow(cuda_device):
    x = torch.randn(1, 64, 32, device=cuda_device).to(torch.bfloat16).requires_grad_(True)
    w = torch.full((32,), 1e4, device=cuda_device)
    y = group_norm(x, 4, w, activation="silu")
    y.backward(torch.ones_like(y))
    r = reference(x.detach(), 4, w, None, 1e-5, True, torch.ones_like(y))
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(x.grad).all())
    assert bool(((y.detach().double() - r["y"]).abs() <= BF16 * r["y"].abs() + FP32 * r["size_h"]).all())


@pytest.mark.parametrize("shape", [(2, 100, 128, 32), (1, 33, 640, 32), (3, 5, 2560, 4), (1, 1, 256, 1)])
def test_codes_are_those_of_the_output(cuda_device, shape):
    x, w, b, dy = inputs(shape, cuda_device, torch.bfloat16)
    a, c = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y, q = group_norm_fp8(a, shape[3], w, b, activation="silu")
    plain = group_norm(c, shape[3], w, b, activation="silu")
    want = quantize_fp8(y.detach())
    assert torch.equal(y, plain) and torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
    y.backward(dy)
    plain.backward(dy)
    assert torch.equal(a.grad, c.grad)


def test_unaligned_tensors_and_what_lies_behind(cuda_device):
    x, w, b, _ = inputs((2, 30, 64, 8), cuda_device, torch.float32)
    want = group_norm(x, 8, w, b)
    for skip in (1, 2, 4):      # elements: 2, 4 and 8 bytes off a 16-byte boundary
        base = torch.empty(x.numel() + skip, dtype=torch.bfloat16, device=cuda_device)
        base[skip:] = x.view(-1)
        got = group_norm(base[skip:].view(x.shape), 8, w, b)
        # other chunks and thread shapes: the statistics may differ in their last bits, an output by one BF16 step
        assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -14)
    n = x.numel()
    y = torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device=cuda_device)
    stats = torch.full((2 * 8 * 2 + 8,), 7.0, device=cuda_device)
    lib = _lib.lib()
    size = lib.flame_group_norm_workspace_bytes(2, 30, 64, 8, 0)
    ws = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device=cuda_device)
    assert lib.flame_group_norm(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), None, None, stats.data_ptr(), 2, 30, 64, 8, 1e-5, 0, 1, ws.data_ptr(), size,
                                torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y[:n].view(x.shape), want) and bool((y[n:] == 7).all()) and bool((stats[32:] == 7).all()) and bool((ws[size:] == 0xAB).all())


def test_views_empty_and_partial_gradients(cuda_device):
    x = torch.randn(2, 16, 8, 12, device=cuda_device).to(memory_format=torch.channels_last).to(torch.bfloat16)
    y = group_norm(x.permute(0, 2, 3, 1), 4)                     # [B, C, H, W] in channels-last memory
    assert torch.equal(y, group_norm(x.permute(0, 2, 3, 1).reshape(2, 96, 16), 4).view(2, 8, 12, 16))
    assert torch.equal(group_norm(x.permute(0, 2, 3, 1).reshape(192, 16), 4), group_norm(x.permute(0, 2, 3, 1).reshape(192, 1, 16), 4).view(192, 16))
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    e = torch.empty(0, 5, 16, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    group_norm(e, 4, w).sum().backward()
    assert e.grad.shape == e.shape and bool((w.grad == 0).all())
    z = torch.empty(3, 0, 16, device=cuda_device, dtype=torch.bfloat16)
    assert group_norm(z, 4).shape == (3, 0, 16)
    t = torch.randn(2, 10, 16, device=cuda_device).to(torch.bfloat16)
    w2, b2 = torch.randn(16, device=cuda_device, requires_grad=True), torch.randn(16, device=cuda_device, requires_grad=True)
    both = torch.autograd.grad(group_norm(t, 4, w2, b2).sum(), (w2, b2))
    assert torch.equal(torch.autograd.grad(group_norm(t, 4, w2, b2.detach()).sum(), w2)[0], both[0])
    assert torch.equal(torch.autograd.grad(group_norm(t, 4, w2.detach(), b2).sum(), b2)[0], both[1])


def test_nonfinite_values_of_narrow_groups(cuda_device):
    """Groups of three channels: pairs and vectors of channels span groups, whose values must not mix."""
    for c, g in ((24, 8), (30, 10), (15, 5)):
        x, w, b, dy = inputs((1, 40, c, g), cuda_device, torch.float32)
        z = x.clone()
        z[0, 7, 4] = float("nan")
        outs = []
        for t in (x, z):
            t = t.requires_grad_(True)
            y = group_norm(t, g, w, b, activation="silu")
            outs.append((y.detach(), torch.autograd.grad(y, t, dy)[0]))
        for clean, got in zip(*outs):
            assert bool(torch.isnan(got[0, :, 3:6]).all())
            keep = [i for i in range(c) if not 3 <= i < 6]
            assert torch.equal(clean[..., keep], got[..., keep])


def test_second_derivatives_are_refused(cuda_device):
    x = torch.randn(1, 8, 16, device=cuda_device).to(torch.bfloat16).requires_grad_(True)
    w = torch.randn(16, 16, device=cuda_device).to(torch.bfloat16)
    for f in (lambda t: group_norm(t, 4), lambda t: fp8_linear(t, w)):
        first = torch.autograd.grad(f(x).float().square().sum(), x, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.float().sum(), x)


def test_same_bits_every_time_on_any_stream_and_in_a_graph(cuda_device):
    x, w, b, dy = inputs((2, 500, 320, 32), cuda_device, torch.float32)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = group_norm(leaves[0], 32, leaves[1], leaves[2], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [step() for _ in range(3)]
    here = [step() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for run in there + here for p, q in zip(run, want))
    graphs = []
    for _ in range(2):       # two graphs, each with workspaces of its own pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    x.copy_(torch.randn(x.shape, device=cuda_device))
    for g, _ in graphs:
        g.replay()
    want = step()
    assert all(torch.equal(p, q) for _, got in graphs for p, q in zip(got, want))


def test_under_a_pool(cuda_device):
    """The tensor the norm saves goes out and comes back: uncompressed, the gradients are the resident ones."""
    x, w, b, dy = inputs((2, 1024, 640, 32), cuda_device, torch.float32)
    lw = (torch.randn(640, 640, device=cuda_device) * 0.04).to(torch.bfloat16)

    def block(t):
        y, q = group_norm_fp8(t, 32, w, b, activation="silu")
        return fp8_linear(y, lw, codes=q)

    def grads(run):
        for p in (w, b, lw):
            p.requires_grad_(True).grad = None
        t = x.clone().requires_grad_(True)
        y = run(t)
        y.backward(dy)
        return [y.detach(), t.grad, w.grad, b.grad, lw.grad]

    want = grads(block)
    pool = ActivationOffloadPool(cuda_device, 8, x.numel() * 2, OffloadCompression.NONE)
    ckpt.set_activation_offload_pool(pool)
    try:
        got = grads(lambda t: ckpt.checkpoint_offload([t], block))
        assert pool.stats()["pushes"] == 2          # the norm's input and the product's
        again = grads(lambda t: ckpt.checkpoint([t], block))
        torch.cuda.synchronize()
    finally:
        ckpt.clear_activation_offload_pool()
        pool.close()
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and all(torch.equal(p, q) for p, q in zip(want, again))


# (batch, positions, channels, groups): slabs of channels that end inside groups, the last one narrower; vectors of two channels and of
# one; as many groups as there may be; parts joined by a launch of their own, groups over several slabs
@pytest.mark.parametrize("shape", [(1, 300, 1280, 32), (1, 40, 1152, 9), (2, 21, 2568, 8), (1, 50, 1030, 10), (1, 30, 771, 3), (1, 9, 8192, 4096), (1, 5000, 4096, 2),
                                   (1, 20000, 1280, 32), (3, 4097, 136, 17)])
def test_ways_to_cut_a_tensor(cuda_device, shape):
    test_output_and_gradients(cuda_device, shape, torch.float32, "silu")


def test_calls_one_behind_the_other(cuda_device):
    """The second launch of a call begins to read x while the first one ends: x changed in place just before, each output the next
    input, and a call's input overwritten just behind it give what they give with pauses between."""
    start = torch.randn(2, 1000, 640, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(7)).to(torch.bfloat16)
    w = torch.full((640,), 1.5, device=cuda_device)

    def run(x, pause):
        outs = []
        for k in range(6):
            x.mul_(1.25).add_(0.5 * k)
            pause()
            y = group_norm(x, 32, w, activation="silu")
            pause()
            z, codes = group_norm_fp8(y, 16, w)
            pause()
            x.copy_(z)
            dx, = torch.autograd.grad(group_norm(y.requires_grad_(True), 32, w), y, z)
            pause()
            outs += [y.detach().clone(), z, codes.dequantize(), dx]
        return outs

    want = run(start.clone(), torch.cuda.synchronize)
    for _ in range(3):
        for a, b in zip(run(start.clone(), lambda: None), want):
            assert torch.equal(a, b)
    x = start.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(x, lambda: None)
    for _ in range(2):
        x.copy_(start)
        graph.replay()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_refusals(cuda_device):
    x = torch.randn(2, 10, 64, device=cuda_device, dtype=torch.bfloat16)
    w = torch.ones(64, device=cuda_device)
    for args, kwargs, text in (((x, 7), {}, "multiple"), ((x, 0), {}, "multiple"), ((x.float(), 8), {}, "BF16"), ((x.transpose(1, 2), 5), {}, "contiguous"),
                               ((x, 8, w[:32]), {}, "weight"), ((x, 8, w, w.bfloat16()), {}, "one type"), ((x, 8, w.double()), {}, "weight"),
                               ((x, 8), {"activation": "gelu"}, "activation"), ((x.cpu(), 8), {}, "on the GPU"), ((x, 8, w.cpu()), {}, "on the GPU|one device")):
        with pytest.raises(InvalidInput, match=text):
            group_norm(*args, **kwargs)
    with pytest.raises(InvalidInput, match="128"):
        group_norm_fp8(x, 8)
    lib = _lib.lib()
    y, stats = torch.empty_like(x), torch.empty(2, 8, 2, device=cuda_device)
    size = lib.flame_group_norm_workspace_bytes(2, 10, 64, 8, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=cuda_device)
    args = [x.data_ptr(), None, None, y.data_ptr(), None, None, stats.data_ptr(), 2, 10, 64, 8, 1e-5, 0, 0, ws.data_ptr(), size, None]
    for at, value, text in ((15, size - 1, "workspace"), (0, None, "null"), (0, x.data_ptr() + 1, "misaligned"), (12, 9, "activation"), (13, 3, "BF16 or F32"), (9, 1 << 20, "channels"), (10, 5000, "multiple")):
        bad = list(args)
        bad[at] = value
        assert lib.flame_group_norm(*bad) == 1 and text in _lib.last_error(), (at, _lib.last_error())
