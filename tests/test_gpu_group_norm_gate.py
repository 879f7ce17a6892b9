"""SiLU of the group norm far below zero, forward and backward: where the gate ends, and what a masked channel's bias leaves behind."""
import pytest
import torch

from flame_b200.group_norm import group_norm, group_norm_fp8

pytestmark = pytest.mark.gpu

# The gate is 0 under h = -60 ln 2 = -41.6, where the formula has 2^-60: the product with h is off by 42 * 2^-60 at most, under 2^-54.
TAIL = 2.0 ** -54
LOWEST = torch.finfo(torch.float32).min


def silu64(h):
    return h * torch.sigmoid(h)


def slope64(h):
    s = torch.sigmoid(h)
    return s * (1 + h * (1 - s))


@pytest.mark.parametrize("channels", [304, 302, 303])      # vectors of eight, two and one
def test_gate_and_its_slope_over_the_range(cuda_device, channels):
    """A weight of zero makes h the bias.  The gate takes an exponential of t = h log2(e), whose rounding is |t| 2^-24 of it at most, and a
    few roundings more: 2^-17 of the value under |t| = 60; then one rounding to BF16, 2^-8.  The slope 1 + h (1 - gate) adds numbers of the
    size of 1 + |h|, and the bias gradient is the sum of `positions` of them."""
    positions = 40
    x = torch.randn(1, positions, channels, device=cuda_device).to(torch.bfloat16)
    w = torch.zeros(channels, device=cuda_device)
    b = torch.linspace(-150, 10, channels, device=cuda_device).requires_grad_(True)
    y = group_norm(x, channels, w, b, activation="silu")
    h = b.detach().double()
    want = silu64(h)
    assert bool(((y.detach().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17 * want.abs() + TAIL).all())
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    size = torch.sigmoid(h) * (1 + h.abs())
    assert bool(((db.double() - positions * slope64(h)).abs() <= positions * (2.0 ** -17 * size + TAIL)).all())


@pytest.mark.parametrize("bias", [-1e4, -1e20, LOWEST])
@pytest.mark.parametrize("channels,groups", [(64, 8), (30, 10), (15, 5)])
def test_a_channel_masked_by_its_bias_is_zero(cuda_device, channels, groups, bias):
    gen = torch.Generator(device=cuda_device).manual_seed(channels)
    n = lambda *s: torch.randn(*s, device=cuda_device, generator=gen)  # noqa: E731
    x, dy = n(2, 50, channels).to(torch.bfloat16), n(2, 50, channels).to(torch.bfloat16)
    w, b = 1 + 0.3 * n(channels), 0.3 * n(channels)
    masked = torch.zeros(channels, dtype=torch.bool, device=cuda_device)
    masked[3::7] = True
    low = torch.where(masked, torch.full_like(b, bias), b)
    leaves = [t.requires_grad_(True) for t in (x, w, low)]
    y = group_norm(x, groups, w, low, activation="silu")
    plain = group_norm(x.detach(), groups, w.detach(), b, activation="silu")
    # Two neighbouring channels share a reciprocal, of the product of their denominators: a gate's last bits depend on its neighbour.  A
    # product (2^-24), the reciprocal (2^-23) and the product with it (2^-24) make 2^-22 of a gate, 2^-21 between two runs, which is one
    # step of BF16 (2^-7) at most.
    assert bool(((y - plain)[..., ~masked].abs() <= 2.0 ** -7 * plain[..., ~masked].abs()).all()) and bool((y[..., masked].abs() <= TAIL).all())
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    # a masked channel passes no gradient on: those of the others are what they are without its output gradient
    some = [t.detach().requires_grad_(True) for t in (x, w, b)]
    rest = torch.where(masked, torch.zeros_like(dy), dy)
    want = torch.autograd.grad(group_norm(some[0], groups, some[1], some[2], activation="silu"), some, rest)
    assert bool((dw[masked].abs() <= 100 * TAIL * 50).all()) and bool((db[masked].abs() <= 100 * TAIL * 50).all())
    # dy gate (1 + h (1 - gate)) errs by 2^-20 of |dy| (1 + |h|) then, and the sums over 100 positions, in either run, by 100 * 2^-24 of
    # the sum of magnitudes: 2^-16 together; the group's sums have up to 500 terms, in chains of a hundred
    g = x.detach().double().view(2, 50, groups, -1)
    rstd = 1 / (g.var((1, 3), keepdim=True, unbiased=False) + 1e-5).sqrt()
    xhat = ((g - g.mean((1, 3), keepdim=True)) * rstd).view(x.shape)
    size = rest.double().abs() * (1 + (xhat * w.detach() + b).abs())
    assert bool(((dw - want[1])[~masked].abs() <= 2.0 ** -16 * (size * xhat.abs()).sum((0, 1))[~masked]).all())
    assert bool(((db - want[2])[~masked].abs() <= 2.0 ** -16 * size.sum((0, 1))[~masked]).all())
    u = (size * w.detach().abs()).view(g.shape)
    size = rstd * (u + u.mean((1, 3), keepdim=True) + xhat.view(g.shape).abs() * (u * xhat.view(g.shape).abs()).mean((1, 3), keepdim=True))
    assert bool(((dx.double() - want[0].double()).abs() <= 2.0 ** -7 * want[0].double().abs() + 2.0 ** -16 * size.view(x.shape)).all())


def test_infinite_biases(cuda_device):
    """-inf times a gate of zero is NaN, as the formula has it; +inf is +inf.  Either stays in its channel."""
    x = torch.randn(1, 50, 64, device=cuda_device).to(torch.bfloat16)
    b = torch.randn(64, device=cuda_device)
    plain = group_norm(x, 8, None, b, activation="silu")
    for value in (float("-inf"), float("inf")):
        low = b.clone()
        low[9] = value
        y = group_norm(x, 8, None, low, activation="silu")
        assert bool(torch.isnan(y[..., 9]).all()) if value < 0 else bool((y[..., 9] == value).all())
        keep = [i for i in range(64) if i != 9]
        assert bool(((y - plain)[..., keep].abs() <= 2.0 ** -7 * plain[..., keep].abs()).all())       # one step, as above


def test_codes_beside_a_masked_channel(cuda_device):
    """A masked channel's output does not decide the scale of its block."""
    x = torch.randn(1, 40, 128, device=cuda_device).to(torch.bfloat16)
    b = torch.zeros(128, device=cuda_device)
    b[5] = LOWEST
    y, q = group_norm_fp8(x, 8, None, b, activation="silu")
    assert bool((y[..., 5].abs() <= TAIL).all()) and bool((q.scales.view(-1) * 448 <= y.float().abs().amax(2).view(-1) * (1 + 2.0 ** -20)).all())
    assert bool((q.scales * 448 < 10).all())
