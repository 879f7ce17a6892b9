"""Cases of the FP8 block product, the channels-last group norm and the counter-based dropout.

``run`` computes them from elementary torch operations, or, where ``own`` is true, through the package's entry points.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token through a projection with frozen FP8 weights: launch latency and the weight bytes
        {"name": "linear, one token", "op": "linear", "m": 1, "k": 2048, "n": 2048},
        # the 77 text tokens of an image model into a four-fold wider layer: few rows, the weight bytes count
        {"name": "linear, 77 tokens", "op": "linear", "m": 77, "k": 2560, "n": 10240},
        # a large batch of tokens with frozen weights: the tensor cores' rate
        {"name": "linear, large", "op": "linear", "m": 8192, "k": 8192, "n": 8192},
        # a training step's linear layer over the image and text tokens of a transformer block: forward, both gradients
        {"name": "linear step", "op": "linear_step", "m": 4608, "k": 2304, "n": 9216},
        # the same with sizes that fill no tile and no block
        {"name": "linear step, ragged", "op": "linear_step", "m": 1000, "k": 1331, "n": 713},
        # the innermost level of an image model, 8 x 8 positions: latency
        {"name": "group norm, 8x8", "op": "norm", "b": 1, "l": 64, "c": 1280, "g": 32, "act": "silu", "params": "float32"},
        # a residual block whose product reads FP8 codes: the norm writes the codes beside its output
        {"name": "group norm, codes", "op": "norm_codes", "b": 2, "l": 4096, "c": 640, "g": 32, "act": "silu", "params": "bfloat16"},
        # the outermost level of an image decoder, 1024 x 1024 positions: larger than the L2 cache
        {"name": "group norm, 1024x1024", "op": "norm", "b": 1, "l": 1048576, "c": 128, "g": 32, "act": "silu", "params": "bfloat16"},
        # a training step's norm at 64 x 64 positions: output and all gradients
        {"name": "group norm step", "op": "norm_step", "b": 4, "l": 4096, "c": 320, "g": 32, "act": "silu", "params": "float32"},
        # odd sizes, no activation
        {"name": "group norm step, odd", "op": "norm_step", "b": 3, "l": 1023, "c": 90, "g": 6, "act": "none", "params": "bfloat16"},
        # a small layer's dropout, output and gradient: latency
        {"name": "dropout step, small", "op": "dropout_step", "rows": 154, "cols": 768, "p": 0.1, "residual": False, "dtype": "bfloat16"},
        # dropout on the hidden states of a transformer block, added to the residual stream: output and gradient
        {"name": "dropout step, residual", "op": "dropout_step", "rows": 9216, "cols": 9216, "p": 0.1, "residual": True, "dtype": "bfloat16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A size spread over the logarithm of the range: half of them multiples of 64, the others as they fall."""
    v = _log(rng, low, high)
    return max(64, v // 64 * 64) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_step", "norm", "norm_codes", "norm_step", "dropout_step"])
    if op in ("linear", "linear_step"):
        most = 8192 ** 3 // (4 if op == "linear_step" else 1)
        while True:
            m = _log(rng, 1, 16384) if op == "linear" else _size(rng, 64, 16384)
            k, n = _size(rng, 64, 12288), _size(rng, 64, 12288)
            if m * k * n <= most:
                return {"op": op, "m": m, "k": k, "n": n}
    if op in ("norm", "norm_codes", "norm_step"):
        most = 1048576 * 128 // (2 if op == "norm_step" else 1)
        while True:
            b, l, g = rng.randint(1, 8), _log(rng, 16, 1048576), rng.choice([1, 4, 8, 16, 32])
            c = g * rng.randint(1, 40)
            if op == "norm_codes":
                c = max(128, c // 128 * 128)
            if c % g == 0 and b * l * c <= most:
                return {"op": op, "b": b, "l": l, "c": c, "g": g, "act": rng.choice(["silu", "silu", "none"]),
                        "params": rng.choice(["float32", "bfloat16"])}
    return {"op": op, "rows": _size(rng, 64, 16384), "cols": _size(rng, 64, 9216), "p": rng.choice([0.05, 0.1, 0.25, 0.5]),
            "residual": rng.random() < 0.5, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}


def _up(n, unit):
    return (n + unit - 1) // unit * unit


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] in ("linear", "linear_step"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = (normal(m, k) * (0.25 + torch.rand(k, device="cuda", generator=g))).to(torch.bfloat16)
        w = normal(n, k).mul_(k ** -0.5).to(torch.bfloat16)
        if case["op"] == "linear":
            # the frozen weight as a program keeps it: codes with rows padded to 16 bytes, a scale for each 128 x 128 tile
            codes, scales = _tile_codes(w)
            s["codes"] = torch.zeros(n, _up(k, 16), dtype=torch.uint8, device="cuda")[:, :k]
            s["codes"].copy_(codes)
            s["scales"] = scales
        else:
            s["w"], s["dy"] = w, (normal(m, n) / m).to(torch.bfloat16)
    elif case["op"] in ("norm", "norm_codes", "norm_step"):
        b, l, c, p = case["b"], case["l"], case["c"], getattr(torch, case["params"])
        x = normal(b, l, c).mul_(0.5 + torch.rand(c, device="cuda", generator=g)).add_(0.5 * normal(c))
        s["x"] = x.to(torch.bfloat16)
        s["weight"], s["bias"] = (1 + 0.2 * normal(c)).to(p), (0.2 * normal(c)).to(p)
        if case["op"] == "norm_step":
            s["dy"] = normal(b, l, c).to(torch.bfloat16)
    else:
        t = getattr(torch, case["dtype"])
        s["x"], s["dy"] = normal(case["rows"], case["cols"]).to(t), normal(case["rows"], case["cols"]).to(t)
        s["base"] = normal(case["rows"], case["cols"]).to(t) if case["residual"] else None
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ (seed * 0x1000193), 7 + (seed << 33)
        s["seed"] &= (1 << 63) - 1
        s["offset"] &= (1 << 63) - 1
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from flame_b200 import dropout, fp8_product, group_norm

    op = s["op"]
    if op == "linear":
        return fp8_product.fp8_linear(s["x"], fp8_product.Fp8Blocks(s["codes"], s["scales"], "tiles"))
    if op == "linear_step":
        x, w = s["x"].detach().requires_grad_(True), s["w"].detach().requires_grad_(True)
        y = fp8_product.fp8_linear(x, w)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), s["dy"])
    if op == "norm":
        return group_norm.group_norm(s["x"], s["g"], s["weight"], s["bias"], eps=1e-5, activation=s["act"])
    if op == "norm_codes":
        y, q = group_norm.group_norm_fp8(s["x"], s["g"], s["weight"], s["bias"], eps=1e-5, activation=s["act"])
        return y, q.dequantize(torch.bfloat16)
    if op == "norm_step":
        x, w, b = (s[k].detach().requires_grad_(True) for k in ("x", "weight", "bias"))
        y = group_norm.group_norm(x, s["g"], w, b, eps=1e-5, activation=s["act"])
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), s["dy"])
    x = s["x"].detach().requires_grad_(True)
    y = dropout.dropout(x, s["p"], seed=s["seed"], offset=s["offset"], residual=s["base"])
    return (y.detach(),) + torch.autograd.grad(y, (x,), s["dy"])


def _run_plain(s):
    op = s["op"]
    if op == "linear":
        k, n = s["k"], s["n"]
        w = s["codes"].view(torch.float8_e4m3fn).float()
        w = w * s["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        return (_row_values(s["x"]) @ w.t()).to(torch.bfloat16)
    if op == "linear_step":
        x, w, dy = s["x"], s["w"], s["dy"]
        codes, scales = _tile_codes(w)
        wq = codes.view(torch.float8_e4m3fn).float() * scales.repeat_interleave(BLOCK, 0)[:s["n"]].repeat_interleave(BLOCK, 1)[:, :s["k"]]
        y = _row_values(x) @ wq.t()
        dx = _row_values(dy) @ wq
        dw = _row_values(dy.t().contiguous()) @ _row_values(x.t().contiguous()).t()
        return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw.to(torch.bfloat16)
    if op in ("norm", "norm_codes", "norm_step"):
        b, l, c, g = s["b"], s["l"], s["c"], s["g"]
        x = s["x"].float().view(b, l, g, c // g)
        mean = x.mean(dim=(1, 3), keepdim=True)
        x = x - mean
        rstd = torch.rsqrt((x * x).mean(dim=(1, 3), keepdim=True) + 1e-5)
        xhat = (x * rstd).view(b, l, c)
        w, beta = s["weight"].float(), s["bias"].float()
        h = xhat * w + beta
        gate = 1 / (1 + torch.exp(-h)) if s["act"] == "silu" else None
        y = (h if gate is None else h * gate).to(torch.bfloat16)
        if op == "norm":
            return y
        if op == "norm_codes":
            return y, _row_values(y.view(b * l, c)).to(torch.bfloat16)
        dh = s["dy"].float()
        if gate is not None:
            dh = dh * gate * (1 + h * (1 - gate))
        db, dw = dh.sum(dim=(0, 1)), (dh * xhat).sum(dim=(0, 1))
        t = (dh * w).view(b, l, g, c // g)
        xh = xhat.view(b, l, g, c // g)
        dx = rstd * (t - t.mean(dim=(1, 3), keepdim=True) - xh * (t * xh).mean(dim=(1, 3), keepdim=True))
        return y, dx.view(b, l, c).to(torch.bfloat16), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)
    x, dy = s["x"], s["dy"]
    keep = (_random_bits(x.numel(), s["seed"], s["offset"], x.device) >= round(s["p"] * 2 ** 32)).view(x.shape)
    scale = 1.0 / (1.0 - s["p"])
    y = torch.where(keep, x.float() * scale, torch.zeros((), device=x.device))
    if s["base"] is not None:
        y = s["base"].float() + y
    return y.to(x.dtype), torch.where(keep, dy.float() * scale, torch.zeros((), device=x.device)).to(x.dtype)


def _padded_blocks(x):
    """[r, c] float32 -> [r, ceil(c/128), 128], zeros behind the last column."""
    r, c = x.shape
    return torch.nn.functional.pad(x, (0, _up(c, BLOCK) - c)).view(r, -1, BLOCK)


def _quotient(top):
    """top / 448 as the nearest binary32 number: by a tensor, since a division by a Python number multiplies by its reciprocal."""
    return top / torch.full_like(top, E4M3_MAX)


def _row_values(x):
    """The values that FP8 codes with a scale for 128 elements of a row stand for."""
    r, c = x.shape
    v = _padded_blocks(x.float())
    scale = _quotient(v.abs().amax(dim=2, keepdim=True))
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1 / scale)
    return ((v * inv).to(torch.float8_e4m3fn).float() * scale).view(r, -1)[:, :c]


def _tile_codes(w):
    """uint8 codes [n, k] and float32 scales [ceil(n/128), ceil(k/128)] of a BF16 weight."""
    n, k = w.shape
    v = torch.nn.functional.pad(w.float(), (0, _up(k, BLOCK) - k, 0, _up(n, BLOCK) - n))
    v = v.view(_up(n, BLOCK) // BLOCK, BLOCK, -1, BLOCK)
    scale = _quotient(v.abs().amax(dim=(1, 3), keepdim=True))
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1 / scale)
    codes = (v * inv).to(torch.float8_e4m3fn).view(torch.uint8).view(_up(n, BLOCK), -1)[:n, :k]
    return codes, scale.view(scale.shape[0], scale.shape[2])


def _philox(c0, c1, c2, c3, seed):
    """Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, SC11) on int64 tensors that hold 32-bit words."""
    mask = 0xFFFFFFFF
    k0, k1 = seed & mask, seed >> 32 & mask
    c2, c3 = torch.full_like(c0, c2), torch.full_like(c0, c3)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & mask) ^ c1 ^ k0, p1 & mask, (p0 >> 32 & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), dim=1)


def _random_bits(n, seed, offset, device):
    """32 random bits for each of n elements: element i takes the 16-bit half i % 8 of block i // 8 as its upper bits, and the
    same half of the block whose counter has bit 63 set as its lower bits."""
    blk = torch.arange((n + 7) // 8, device=device)
    lo, hi = blk & 0xFFFFFFFF, blk >> 32

    def halves(top):
        words = _philox(lo, hi | top, offset & 0xFFFFFFFF, offset >> 32 & 0xFFFFFFFF, seed)
        return torch.stack((words & 0xFFFF, words >> 16), dim=2).view(-1)[:n]

    return halves(0) << 16 | halves(1 << 31)


# ---- work --------------------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("linear", "linear_step"):
        m, k, n = case["m"], case["k"], case["n"]
        if op == "linear":
            tiles = -(-n // BLOCK) * -(-k // BLOCK)
            return {"bytes": 2 * m * k + n * k + 4 * tiles + 2 * m * n, "flops": 2 * m * n * k}
        return {"bytes": 2 * (m * k + n * k + m * n) + 2 * (m * n + m * k + n * k), "flops": 6 * m * n * k}
    if op in ("norm", "norm_codes", "norm_step"):
        e, c = case["b"] * case["l"] * case["c"], case["c"]
        par = 4 if case["params"] == "float32" else 2
        if op == "norm":
            return {"bytes": 4 * e + 2 * par * c, "flops": 12 * e}
        if op == "norm_codes":   # x, y, and the codes' values in BF16
            return {"bytes": 6 * e + 2 * par * c, "flops": 16 * e}
        return {"bytes": 8 * e + 4 * par * c, "flops": 36 * e}
    e, size = case["rows"] * case["cols"], 2 if case["dtype"] == "bfloat16" else 4
    return {"bytes": (5 if case["residual"] else 4) * size * e, "flops": 2 * e}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        w = _decode64(s["codes"]) * _spread64(s["scales"], *s["codes"].shape)
        return _blocks64(s["x"].double(), 1, BLOCK) @ w.T
    if op == "linear_step":
        x, w, dy = (s[k].double() for k in ("x", "w", "dy"))
        wq = _blocks64(w, BLOCK, BLOCK)
        return (_blocks64(x, 1, BLOCK) @ wq.T, _blocks64(dy, 1, BLOCK) @ wq, _blocks64(dy, BLOCK, 1).T @ _blocks64(x, BLOCK, 1))
    if op in ("norm", "norm_codes", "norm_step"):
        b, l, c, g = case["b"], case["l"], case["c"], case["g"]
        x = s["x"].double().view(b, l, g, c // g)
        n = l * (c // g)
        mu = x.sum((1, 3), keepdim=True) / n
        sd = (((x - mu) ** 2).sum((1, 3), keepdim=True) / n + 1e-5).sqrt()
        z = ((x - mu) / sd).reshape(b, l, c)
        del x
        w = s["weight"].double()
        h = z * w + s["bias"].double()
        silu = case["act"] == "silu"
        y = h * torch.sigmoid(h) if silu else h
        if op == "norm":
            return y
        if op == "norm_codes":
            # the codes are those of the BF16 output
            return y, _blocks64(y.to(torch.bfloat16).double().view(b * l, c), 1, BLOCK)
        q = torch.sigmoid(h)
        dh = s["dy"].double() * (q + h * q * (1 - q)) if silu else s["dy"].double()
        u = (dh * w).view(b, l, g, c // g)
        zg = z.view(b, l, g, c // g)
        dx = (u - u.sum((1, 3), keepdim=True) / n - zg * ((u * zg).sum((1, 3), keepdim=True) / n)) / sd
        return y, dx.reshape(b, l, c), (dh * z).sum((0, 1)), dh.sum((0, 1))
    x, dy = s["x"].double(), s["dy"].double()
    keep = torch.from_numpy(_keep_numpy(x.numel(), s["seed"], s["offset"], case["p"])).to(x.device).view(x.shape)
    y = torch.zeros_like(x)
    y[keep] = x[keep] / (1 - case["p"])
    dx = torch.zeros_like(dy)
    dx[keep] = dy[keep] / (1 - case["p"])
    return (y if s["base"] is None else y + s["base"].double()), dx


def _decode64(codes):
    """E4M3 codes: sign, four exponent bits with bias 7, three mantissa bits; exponent 0 holds multiples of 2^-9."""
    c = codes.to(torch.int64)
    e, f = (c >> 3 & 15).double(), (c & 7).double()
    v = torch.where(e == 0, f / 512, (1 + f / 8) * torch.exp2(e - 7))
    return torch.where(c >= 128, -v, v)


def _spread64(scales, rows, cols):
    i, j = torch.arange(rows, device=scales.device) // BLOCK, torch.arange(cols, device=scales.device) // BLOCK
    return scales.double()[i][:, j]


def _blocks64(v, down, across):
    """The values of E4M3 codes with one scale for each `down` x `across` block of a matrix of doubles.  The codec defines the
    scale, its reciprocal and the product that is encoded as binary32 numbers; each is rounded to that here."""
    r, c = v.shape
    rr, cc = _up(r, down), _up(c, across)
    out = torch.zeros(rr, cc, dtype=torch.float64, device=v.device)
    out[:r, :c] = v
    t = out.view(rr // down, down, cc // across, across)
    top = t.abs().amax((1, 3), keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), (top / E4M3_MAX).float().double())
    t = (t * (1 / scale).float().double()).float().double()
    # to the nearest multiple of the code's step, ties to the even one: 2^(e - 3) in [2^e, 2^(e+1)), 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    t = (torch.round(t / step) * step).clamp(-E4M3_MAX, E4M3_MAX) * scale
    return t.reshape(rr, cc)[:r, :c].contiguous()


def _keep_numpy(n, seed, offset, p):
    out = np.empty(n, dtype=bool)
    chunk = 1 << 22          # elements at a time, a multiple of 8
    low = np.uint64(0xFFFFFFFF)
    for first in range(0, n, chunk):
        count = min(chunk, n - first)
        blk = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
        parts = []
        for top in (0, 1 << 31):
            c = [blk & low, blk >> np.uint64(32) | np.uint64(top), np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32 & 0xFFFFFFFF)]
            k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
            for _ in range(10):
                a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
                c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
                k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
            parts.append(np.stack(c, axis=1).astype("<u4").view("<u2").reshape(-1)[:count].astype(np.uint64))
        u = parts[0] << np.uint64(16) | parts[1]
        out[first:first + count] = u >= np.uint64(round(p * 2 ** 32))
    return out
