"""What is measured of the 8-bit operators: activation checkpoints in 8 bits and products of 8-bit blocks.

The format: a row's values in blocks of 128 (the last may be shorter); a block has one scale 2^e, e the smallest integer >= -126 with
max |x| <= F 2^e (F = 448 for e4m3, 57344 for e5m2), and its codes are x 2^-e rounded to nearest even.

  save8       an activation saved in 8 bits and restored
  linear8     y = Q(x) W8^T + bias, W8 kept in 8 bits: the product of a serving path
  train8      the same layer in training: y, and the gradients of x, w and bias from the checkpoint Q(x)
  an_relu8    the coupling networks' ActNorm + ReLU: y, and the gradients of x, bias and logs from its checkpoint
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
# per format: torch's type, mantissa bits, exponent of the smallest normal value, exponent of the largest (1.75 2^top)
FORMATS = {"e4m3": (torch.float8_e4m3fn, 3, -6, 8), "e5m2": (torch.float8_e5m2, 2, -14, 15)}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one pixel's 320 conditioning channels: latency only
        {"name": "save8 one pixel", "op": "save8", "rows": 1, "cols": 320, "dtype": "f32", "fmt": "e4m3"},
        # the coupling networks' 64 hidden channels of 8 planes of 80 x 80
        {"name": "save8 hidden planes", "op": "save8", "rows": 51200, "cols": 64, "dtype": "f32", "fmt": "e4m3"},
        # odd row length, gradients' wider range
        {"name": "save8 ragged", "op": "save8", "rows": 6401, "cols": 333, "dtype": "f16", "fmt": "e5m2"},
        # a long batch of wide activations
        {"name": "save8 large", "op": "save8", "rows": 32768, "cols": 4096, "dtype": "bf16", "fmt": "e4m3"},
        # a single row through a large layer: the weights' bytes
        {"name": "linear8 one row", "op": "linear8", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": True},
        # a few rows, nothing a multiple of a tile
        {"name": "linear8 few ragged rows", "op": "linear8", "m": 13, "n": 2049, "k": 1000, "dtype": "f16", "bias": True},
        # an ordinary batch
        {"name": "linear8 batch", "op": "linear8", "m": 512, "n": 2048, "k": 2048, "dtype": "bf16", "bias": True},
        # a long batch: bound by the matrix cores
        {"name": "linear8 large", "op": "linear8", "m": 8192, "n": 8192, "k": 4096, "dtype": "bf16", "bias": False},
        # a per-pixel layer 320 -> 64 over 8 planes of 20 x 20 + 1
        {"name": "train8 pixels", "op": "train8", "m": 3201, "n": 64, "k": 320, "dtype": "f32", "bias": True},
        # a wide layer in bf16
        {"name": "train8 large", "op": "train8", "m": 16384, "n": 2048, "k": 2048, "dtype": "bf16", "bias": True},
        # the smallest hidden plane, and the first level of 512 x 512 patches
        {"name": "an_relu8 small", "op": "an_relu8", "b": 1, "h": 10, "w": 10, "c": 64},
        {"name": "an_relu8 large", "op": "an_relu8", "b": 8, "h": 256, "w": 256, "c": 64},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["save8", "linear8", "train8", "an_relu8"])
    if op == "save8":
        cols = _log(rng, 1, 8192)
        return {"op": op, "rows": _log(rng, 1, min(65536, 100_000_000 // cols)), "cols": cols, "dtype": rng.choice(sorted(DTYPES)), "fmt": rng.choice(sorted(FORMATS))}
    if op == "linear8":
        n, k = _log(rng, 16, 8192), _log(rng, 32, 8192)
        return {"op": op, "m": _log(rng, 1, min(8192, 250_000_000_000 // (n * k))), "n": n, "k": k, "dtype": rng.choice(sorted(DTYPES)), "bias": rng.random() < 0.5}
    if op == "train8":
        n, k = _log(rng, 16, 4096), _log(rng, 16, 4096)
        return {"op": op, "m": _log(rng, 16, min(32768, 60_000_000_000 // (n * k))), "n": n, "k": k, "dtype": rng.choice(sorted(DTYPES)), "bias": rng.random() < 0.5}
    c, b = rng.choice([32, 64, 96, 128, 320]), rng.randint(1, 16)
    side = int(math.sqrt(30_000_000 / (b * c)))
    return {"op": op, "b": b, "h": _log(rng, 4, min(256, side)), "w": _log(rng, 4, min(256, side)), "c": c}


def work(case):
    """Inputs once, outputs once, and the checkpoint written once and read once: keeping it is what these operators are for."""
    op = case["op"]
    if op == "save8":
        r, c, e = case["rows"], case["cols"], SIZE[case["dtype"]]
        return {"bytes": 2 * r * c * e + 2 * r * (c + -(-c // 128)), "flops": 6 * r * c}
    if op == "linear8":
        m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
        return {"bytes": m * k * e + n * (k + -(-k // 128)) + m * n * e + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "train8":
        m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
        return {"bytes": e * (2 * m * k + 2 * m * n + 2 * n * k + (2 * n if case["bias"] else 0)) + 2 * m * (k + -(-k // 128)), "flops": 6 * m * n * k}
    px, c = case["b"] * case["h"] * case["w"], case["c"]
    return {"bytes": 4 * 4 * px * c + 2 * px * (c + -(-c // 128)) + 16 * c, "flops": 12 * px * c}


# ------------------------------------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """Normal values whose spread differs by channel and by row, with a few far outliers, as activations have it."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(1, cols, generator=g, device="cuda")) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    far = torch.rand(rows, cols, generator=g, device="cuda") < 1e-3
    return torch.where(far, 20 * x, x).to(dtype)


def _ring(x):
    return torch.nn.functional.pad(x, (0, 0, 1, 1, 1, 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op == "save8":
        return {**case, "x": _activations(g, case["rows"], case["cols"], DTYPES[case["dtype"]])}
    if op == "an_relu8":
        b, h, w, c = case["b"], case["h"], case["w"], case["c"]
        s = {**case, "x": _ring(_activations(g, b * h * w, c, torch.float32).view(b, h, w, c))}
        s["grad"] = _ring(0.01 * torch.randn(b, h, w, c, generator=g, device="cuda"))
        s["bias"] = 0.5 * torch.randn(c, generator=g, device="cuda")
        s["logs"] = 0.3 * torch.randn(c, generator=g, device="cuda")
        return s
    m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
    s = {**case, "x": _activations(g, m, k, dtype)}
    w = torch.randn(n, k, generator=g, device="cuda") * (torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda")) / math.sqrt(k))
    s["bias"] = (0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype) if case["bias"] else None
    if op == "train8":
        s["w"] = w.to(dtype)
        s["grad"] = (0.01 * _activations(g, m, n, torch.float32)).to(dtype)
        return s
    # a serving program keeps its weights in 8 bits: the codes in rows of whole 16 bytes, the scales' exponents as bytes
    values, exponents = _split8(w, "e4m3")
    codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    codes[:, :k] = values.to(torch.float8_e4m3fn)
    scales = torch.zeros(n, -(-k // 512) * 4, dtype=torch.uint8, device="cuda")
    scales[:, : exponents.shape[1]] = (exponents + 127).to(torch.uint8)
    s["codes"], s["scales"] = codes[:, :k], scales.view(torch.float8_e8m0fnu)[:, : exponents.shape[1]]
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _power(e):
    """2^e in float32, e from -126 to 127, by its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _split8(x, fmt):
    """(codes' values, blocks' exponents): x in blocks of 128 along its rows."""
    _, bits, low, top = FORMATS[fmt]
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % 128)).view(rows, -1, 128)
    m = torch.where(x.isfinite(), x.abs(), 0.0).amax(2)
    # the exponent of m, one more where its mantissa is over 1.75
    e = (((m.view(torch.int32) + 0x1FFFFF) >> 23) - 127 - top).clamp(min=-126)
    v = x * _power(-e)[:, :, None]
    step = (((v.view(torch.int32) >> 23) & 255) - 127).clamp(min=low, max=127) - bits
    v = torch.round(v * _power(-step)) * _power(step)
    if fmt == "e4m3":
        v = torch.where(v.isinf(), math.nan, v)
    return v.view(rows, -1)[:, :cols], e


def _join8(v, e):
    """The float32 values that codes and exponents stand for."""
    return v * _power(e).repeat_interleave(128, dim=1)[:, : v.shape[1]]


def _q8(x, fmt="e4m3"):
    return _join8(*_split8(x, fmt))


def _plain(s):
    op = s["op"]
    if op == "save8":
        return _q8(s["x"], s["fmt"]).to(s["x"].dtype)
    if op == "an_relu8":
        x, g = s["x"][:, 1:-1, 1:-1], s["grad"][:, 1:-1, 1:-1]
        scale = torch.exp(s["logs"])
        v = (x + s["bias"]).clamp(min=0)
        q, e = _split8(v.reshape(-1, s["c"]), "e4m3")
        q = torch.where((q == 0) & (v.reshape(q.shape) > 0), 2.0 ** -9, q)      # a positive value stays one: the mask is exact
        q = _join8(q, e).view(v.shape)
        g = torch.where(q != 0, g, 0.0)
        return {"y": _ring(v * scale), "dx": _ring(g * scale), "dbias": scale * g.sum((0, 1, 2)), "dlogs": scale * (g * q).sum((0, 1, 2))}
    x, dtype = s["x"], s["x"].dtype
    q = _q8(x)
    if op == "linear8":
        w = _join8(s["codes"].float(), s["scales"].view(torch.uint8).int() - 127)
        y = q @ w.t()
        return (y + s["bias"].float() if s["bias"] is not None else y).to(dtype)
    w, g = s["w"], s["grad"]
    y = q @ _q8(w).t()
    out = {"y": (y + s["bias"].float() if s["bias"] is not None else y).to(dtype)}
    out["dx"] = (_q8(g) @ _q8(w.t()).t()).to(dtype)
    out["dw"] = (g.float().t() @ q).to(dtype)
    if s["bias"] is not None:
        out["dbias"] = g.float().sum(0).to(dtype)
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _framework(s):
    from interflow_amd import block8, train_ops

    op = s["op"]
    if op == "save8":
        return block8.dequantize(block8.quantize(s["x"], s["fmt"]), s["x"].dtype)
    if op == "linear8":
        return block8.linear(s["x"], block8.Block8(s["codes"], s["scales"]), s["bias"])
    x = s["x"].detach().requires_grad_()
    if op == "an_relu8":
        bias, logs = s["bias"].detach().requires_grad_(), s["logs"].detach().requires_grad_()
        y, _ = train_ops.an_relu8_ring(x, bias, logs)
        dx, dbias, dlogs = torch.autograd.grad(y, (x, bias, logs), s["grad"])
        return {"y": y.detach(), "dx": dx, "dbias": dbias, "dlogs": dlogs}
    w = s["w"].detach().requires_grad_()
    if s["bias"] is None:
        y = train_ops.linear8(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), s["grad"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    bias = s["bias"].detach().requires_grad_()
    y = train_ops.linear8(x, w, bias)
    dx, dw, dbias = torch.autograd.grad(y, (x, w, bias), s["grad"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "dbias": dbias}


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _two_to(e):
    """2^e in float64 by its bits (a library's pow is off by a last bit, and ties between codes would go another way)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact8(x, fmt, keep_positive=False):
    """The values that x's rows have in 8 bits, in float64, from the format's definition; inputs are finite."""
    _, bits, low, top = FORMATS[fmt]
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], 128):
        b = x[:, at:at + 128]
        f, q = torch.frexp(b.abs().amax(1, keepdim=True))              # m = f 2^q, 0.5 <= f < 1: m <= 1.75 2^(q-1) where f <= 0.875
        e = (q - 1 - top + (f > 0.875).int()).clamp(min=-126)
        v = b * _two_to(-e)
        _, q = torch.frexp(v)
        step = _two_to((q - 1).clamp(min=low) - bits)
        r = torch.round(v / step) * step
        if keep_positive:
            r = torch.where((r == 0) & (v > 0), 2.0 ** (low - bits), r)
        out[:, at:at + 128] = r * _two_to(e)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "save8":
        return _exact8(s["x"], s["fmt"])
    if op == "an_relu8":
        c = case["c"]
        x, g = s["x"][:, 1:-1, 1:-1].double(), s["grad"][:, 1:-1, 1:-1].double()
        scale = s["logs"].double().exp()
        # what is saved is the float32 sum x + bias: it decides which way a value between two codes goes
        v = (x + s["bias"].double()).float().double().relu()
        q = _exact8(v.reshape(-1, c), "e4m3", keep_positive=True).view(v.shape)
        g = g * (v > 0)
        return {"y": _ring((x + s["bias"].double()).relu() * scale), "dx": _ring(g * scale), "dbias": scale * g.sum((0, 1, 2)), "dlogs": scale * (g * q).sum((0, 1, 2))}
    q = _exact8(s["x"], "e4m3")
    bias = s["bias"].double() if s["bias"] is not None else 0.0
    if op == "linear8":
        scales = _two_to(s["scales"].view(torch.uint8).int() - 127)
        w = s["codes"].double() * scales[:, torch.arange(case["k"], device="cuda") // 128]
        return q @ w.t() + bias
    w, g = s["w"], s["grad"].double()
    out = {"y": q @ _exact8(w, "e4m3").t() + bias, "dx": _exact8(g, "e4m3") @ _exact8(w.t(), "e4m3").t(), "dw": g.t() @ q}
    if s["bias"] is not None:
        out["dbias"] = g.sum(0)
    return out
