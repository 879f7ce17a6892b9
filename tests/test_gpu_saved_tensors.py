"""The operators under saved-tensor hooks that give a saved tensor back in other memory, with another stride, or from the host."""
import pytest
import torch

from flame_b200.dropout import dropout
from flame_b200.fp8_product import fp8_linear, quantize_fp8
from flame_b200.group_norm import group_norm

pytestmark = pytest.mark.gpu


def elsewhere(t):
    """The same numbers with every row of the last dimension behind a gap."""
    if t.dim() == 0:
        return t.clone()
    base = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    out = base[..., 1:1 + 2 * t.shape[-1]:2]
    out.copy_(t)
    return out


def hooks():
    yield torch.autograd.graph.save_on_cpu()
    yield torch.autograd.graph.save_on_cpu(pin_memory=True)
    yield torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)
    yield torch.autograd.graph.saved_tensors_hooks(elsewhere, lambda t: t)


@pytest.mark.parametrize("m,n,k", [(5, 48, 64), (33, 130, 1331), (70, 257, 129), (4, 1, 20)])
def test_linear_layers(cuda_device, m, n, k):
    g = torch.Generator(device=cuda_device).manual_seed(m + n + k)
    x, w, dy = (torch.randn(s, device=cuda_device, generator=g).to(torch.bfloat16) for s in ((m, k), (n, k), (m, n)))
    frozen = quantize_fp8(w, "tiles")
    wide = torch.randn(m, k + 24, device=cuda_device, generator=g).to(torch.bfloat16)
    wide[:, 8:8 + k] = x
    for source in (x, wide[:, 8:8 + k], x.view(1, m, k)):
        for weight in (frozen, w):
            def step():
                a = source.detach().requires_grad_(True)
                leaves = [a] if weight is frozen else [a, weight.detach().requires_grad_(True)]
                return leaves, fp8_linear(a, frozen if weight is frozen else leaves[1])

            leaves, y = step()
            want = torch.autograd.grad(y, leaves, dy.view(y.shape))
            for hook in hooks():
                with hook:
                    leaves, y = step()
                got = torch.autograd.grad(y, leaves, dy.view(y.shape))
                assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("shape,groups", [((2, 40, 64), 8), ((3, 7, 9, 90), 6), ((1, 5, 15), 5)])
def test_group_norm_and_dropout(cuda_device, shape, groups):
    g = torch.Generator(device=cuda_device).manual_seed(shape[1])
    n = lambda *s: torch.randn(*s, device=cuda_device, generator=g)  # noqa: E731
    x, dy = n(*shape).to(torch.bfloat16), n(*shape).to(torch.bfloat16)
    w, b = 1 + 0.3 * n(shape[-1]), 0.3 * n(shape[-1])
    seed = torch.tensor([5], device=cuda_device)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        return leaves, dropout(group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu"), 0.2, seed=seed, offset=1)

    leaves, y = step()
    want = torch.autograd.grad(y, leaves, dy)
    for hook in hooks():
        with hook:
            leaves, y = step()
        got = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
