"""The operators as a model uses them: a residual block of an image model in channels-last tokens, and a transformer block."""
import pytest
import torch

from flame_b200 import ActivationOffloadPool, OffloadCompression
from flame_b200 import checkpoint as ckpt
from flame_b200 import dit_workload as W
from flame_b200.dropout import dropout
from flame_b200.fp8_product import fp8_linear, quantize_fp8
from flame_b200.group_norm import group_norm, group_norm_fp8

pytestmark = pytest.mark.gpu


class Residual(torch.nn.Module):
    """x + product(dropout(product(silu(group norm(x)))))"""

    def __init__(self, channels, device):
        super().__init__()
        g = torch.Generator(device=device).manual_seed(4)
        n = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
        self.norm_w, self.norm_b = torch.nn.Parameter(1 + 0.1 * n(channels)), torch.nn.Parameter(0.1 * n(channels))
        self.up = torch.nn.Parameter((n(2 * channels, channels) * channels ** -0.5).to(torch.bfloat16))
        self.down = torch.nn.Parameter((n(channels, 2 * channels) * (2 * channels) ** -0.5).to(torch.bfloat16))

    def forward(self, x):
        y, codes = group_norm_fp8(x, 32, self.norm_w, self.norm_b, activation="silu")
        h = dropout(fp8_linear(y, self.up, codes=codes), 0.1, seed=11, offset=0)
        return dropout(fp8_linear(h, self.down), 0.1, seed=11, offset=1, residual=x)


def grads(model, x, dy, run):
    for p in model.parameters():
        p.grad = None
    t = x.clone().requires_grad_(True)
    y = run(t)
    y.backward(dy)
    return [y.detach(), t.grad, *(p.grad.clone() for p in model.parameters())]


def test_residual_block_resident_recomputed_and_offloaded(cuda_device):
    """The same bits whether the block's activations stay, are recomputed (the masks are drawn again) or go out and come back."""
    model = Residual(256, cuda_device)
    x = torch.randn(2, 1024, 256, device=cuda_device).to(torch.bfloat16)
    dy = torch.randn_like(x)
    want = grads(model, x, dy, model)
    assert all(torch.isfinite(t).all() for t in want)
    got = grads(model, x, dy, lambda t: ckpt.checkpoint([t], model))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    pool = ActivationOffloadPool(cuda_device, 8, 4 * x.numel() * 2, OffloadCompression.NONE)
    ckpt.set_activation_offload_pool(pool)
    try:
        for _ in range(2):
            got = grads(model, x, dy, lambda t: ckpt.checkpoint_offload([t], model, min_bytes=1 << 16))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert pool.stats()["pushes"] >= 6       # the norm's input and both products'
    finally:
        ckpt.clear_activation_offload_pool()
        pool.close()


def test_residual_block_against_its_parts_in_64_bits(cuda_device):
    """Each step's output from the step before it in 64 bits: the whole is the chain of its parts.  An element errs by one rounding to BF16
    (2^-8), the products and the norm by 2^-14 of the largest value beside that."""
    model = Residual(128, cuda_device)
    x = torch.randn(1, 300, 128, device=cuda_device).to(torch.bfloat16)
    with torch.no_grad():
        y, codes = group_norm_fp8(x, 32, model.norm_w, model.norm_b, activation="silu")
        g = x.double().view(1, 300, 32, 4)
        h = (g - g.mean((1, 3), keepdim=True)) / (g.var((1, 3), keepdim=True, unbiased=False) + 1e-5).sqrt()
        h = h.view(1, 300, 128) * model.norm_w.double() + model.norm_b.double()
        steps = [(y, h * torch.sigmoid(h))]
        u = fp8_linear(y, model.up, codes=codes)
        steps.append((u, (codes.dequantize().double() @ quantize_fp8(model.up, "tiles").dequantize().double().T).view(1, 300, 256)))
        d = dropout(u, 0.1, seed=11, offset=0)
        keep = dropout(torch.ones_like(u, dtype=torch.float32), 0.1, seed=11, offset=0) != 0
        steps.append((d, torch.where(keep, u.double() / 0.9, torch.zeros((), dtype=torch.float64, device=cuda_device))))
        v = fp8_linear(d, model.down)
        steps.append((v, quantize_fp8(d).dequantize().double().view(1, 300, 256) @ quantize_fp8(model.down, "tiles").dequantize().double().T))
        keep = dropout(torch.ones_like(v, dtype=torch.float32), 0.1, seed=11, offset=1) != 0
        z = dropout(v, 0.1, seed=11, offset=1, residual=x)
        steps.append((z, x.double() + torch.where(keep, v.double() / 0.9, torch.zeros((), dtype=torch.float64, device=cuda_device))))
        for got, want in steps:
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * want.abs().max()).all())
        assert torch.equal(model(x), z)


def test_two_streams_at_once(cuda_device):
    """Steps of different sizes, issued in turn on two streams, give what they give one after the other."""
    jobs = []
    for k, (channels, positions) in enumerate(((256, 3000), (640, 700))):
        model = Residual(channels, cuda_device)
        x = torch.randn(2, positions, channels, device=cuda_device).to(torch.bfloat16)
        jobs.append((model, x, torch.randn_like(x), torch.cuda.Stream()))

    def step(model, x, dy):
        t = x.detach().requires_grad_(True)
        y = model(t)
        return [y.detach(), *torch.autograd.grad(y, [t, *model.parameters()], dy)]

    want = [step(*job[:3]) for job in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for job in jobs:
            with torch.cuda.stream(job[3]):
                got.append(step(*job[:3]))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))


def test_a_recorded_step_with_a_seed_in_device_memory(cuda_device):
    """Norm, product and dropout, forward and backward, in one graph; each replay draws the mask of the seed it finds."""
    x = torch.randn(1, 512, 128, device=cuda_device).to(torch.bfloat16)
    dy = torch.randn_like(x)
    w, nw = (torch.randn(128, 128, device=cuda_device) * 0.1).to(torch.bfloat16), torch.ones(128, device=cuda_device)
    seed = torch.tensor([3], device=cuda_device)

    def step(s):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, nw)]
        y = dropout(fp8_linear(group_norm(leaves[0], 8, leaves[2], activation="silu"), leaves[1]), 0.2, seed=s, offset=4, residual=leaves[0])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    step(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(seed)
    for value in (3, 9):
        seed.fill_(value)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step(value)))


def test_transformer_block_in_fp8_with_dropout(cuda_device):
    """The workload's block with its products in FP8 and residual dropout: resident, recomputed and offloaded agree (the attention's
    backward is not bit-reproducible from run to run, everything else is)."""
    torch.manual_seed(0)
    blk = W.DiTBlock(3).to(cuda_device, torch.bfloat16)
    x = torch.randn(1, W.TOKENS, W.HIDDEN, device=cuda_device, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    cos, sin = W.rope_tables(cuda_device)
    rel = lambda a, b: float((a.detach().float() - b.detach().float()).norm() / a.detach().float().norm().clamp_min(1e-30))  # noqa: E731
    plain = blk(x, cos, sin)
    try:
        W.FP8_LINEARS = True
        fp8 = blk(x, cos, sin)
        # a rounding to e4m3 is off by 2^-4 of the value at most, and the branches are not larger than the residual stream here
        assert 0 < rel(plain, fp8) < 2.0 ** -4
        W.DROPOUT_P, W.DROPOUT_SEED = 0.1, 5
        want = grads(blk, x, dy, lambda t: blk(t, cos, sin))
        got = grads(blk, x, dy, lambda t: ckpt.checkpoint([t, cos, sin], blk))
        assert torch.equal(want[0], got[0]) and max(rel(a, b) for a, b in zip(want, got)) < 5e-3
        saved = ckpt.saved_bytes_of(blk, [x.detach().requires_grad_(True), cos, sin])
        pool = ActivationOffloadPool(cuda_device, 16, saved, OffloadCompression.NONE)
        ckpt.set_activation_offload_pool(pool)
        got = grads(blk, x, dy, lambda t: ckpt.checkpoint_offload([t, cos, sin], blk))
        torch.cuda.synchronize()
        ckpt.clear_activation_offload_pool()
        pool.close()
        assert torch.equal(want[0], got[0]) and max(rel(a, b) for a, b in zip(want, got)) < 5e-3
        W.DROPOUT_SEED = 6
        assert not torch.equal(blk(x, cos, sin), want[0])
    finally:
        W.FP8_LINEARS, W.DROPOUT_P, W.DROPOUT_SEED = False, 0.0, 0
        ckpt.clear_activation_offload_pool()
