"""Gradients of groups without a spread (a blank patch), whose values are far from zero."""
import pytest
import torch

from flame_b200.group_norm import group_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels,groups", [(64, 8), (30, 10), (15, 5), (1280, 32)])
@pytest.mark.parametrize("activation", ["silu", None])
def test_gradients_of_constant_groups(cuda_device, channels, groups, activation):
    """x - mean is exactly 0 there, so h is the bias, rstd is 1/sqrt(eps) and dx = rstd (w dh - mean of w dh).  An element takes a dozen
    binary32 roundings of those terms and sums of 50 x C/G of them in chains of a hundred at most: 2^-16 of their magnitudes, which do
    not grow with the mean; then one rounding to BF16, 2^-8 of the value."""
    gen = torch.Generator(device=cuda_device).manual_seed(channels + groups)
    n = lambda *s: torch.randn(*s, device=cuda_device, generator=gen)  # noqa: E731
    values = torch.tensor([0.0, 3.0, -200.0, 1000.0, 9984.0, -30000.0, 2.0 ** 20], device=cuda_device).to(torch.bfloat16)
    cg, eps = channels // groups, 1e-5
    x = torch.stack([values[(torch.arange(groups, device=cuda_device) + i) % len(values)].repeat_interleave(cg).expand(50, channels) for i in range(3)]).contiguous()
    w, b, dy = 1 + 0.3 * n(channels), 0.5 + 0.3 * n(channels), n(3, 50, channels).to(torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = group_norm(x, groups, w, b, eps=eps, activation=activation)
    h = b.detach().double().expand(3, 50, channels)
    s = torch.sigmoid(h)
    want = h * s if activation else h
    assert bool(((y.detach().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -16) * want.abs()).all())
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    dh = dy.double() * (s * (1 + h * (1 - s)) if activation else 1.0)
    u = (dh * w.detach().double()).view(3, 50, groups, cg)
    rstd = 1 / eps ** 0.5
    want = rstd * (u - u.mean((1, 3), keepdim=True))
    size = rstd * (u.abs() + u.abs().mean((1, 3), keepdim=True))
    got = dx.double().view(want.shape)
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * size).all())
    assert bool((dw == 0).all())
    assert bool(((db.double() - dh.sum((0, 1))).abs() <= 2.0 ** -16 * dh.abs().sum((0, 1))).all())
