"""The 8-bit operators on the GPU against float64: quantize / dequantize bit for bit, products, weight gradients, the linear layer
and ActNorm + ReLU with 8-bit checkpoints, and the training path that uses them.

Tolerances: a float32 sum of n products p has an error of at most n 2^-23 sum |p| (each addition loses less than one unit of the
last of 24 places of a partial sum that is at most sum |p|), and an output of type t is off by half a step more,
finfo(t).eps / 2 of its value (float16: or half its smallest subnormal).  A bfloat16 or float16 result of the matrix product comes from
the 8-bit matrix instructions, which among 8 products drop what is below 2^-13 of the largest: at most 7 * 2^-13 sum |p| more."""
import math

import pytest
import torch

from interflow_amd import block8, hip, train_flow, train_ops
from tests import _block8_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(g, *shape, spread=0.0, dtype=torch.float32):
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn(*shape, generator=g))
    return x.to(dtype).cuda()


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    """Equal values, NaN in the same places (a float16 input of these tests overflows here and there)."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def close(got, ref, n, mag, what="", product8=False):
    """got against ref (float64): a float32 sum of n products whose magnitudes add up to mag, rounded once to got's type."""
    fi = torch.finfo(got.dtype)
    err = n * 2.0 ** -23 * mag
    if product8 and got.dtype != torch.float32:
        err = err + 7 * 2.0 ** -13 * mag
    tol = err + fi.eps / 2 * (ref.abs() + err) + fi.tiny * fi.eps / 2
    over = (got.double() - ref).abs() > tol
    bad = over & (ref.abs() <= fi.max)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - ref).abs() / tol)[bad].max()))


# ------------------------------------------------------------------------------------------------ quantize, dequantize
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 320), (3, 7), (5, 32), (130, 33), (64, 64), (67, 100), (1000, 128), (9, 129), (33, 333), (7, 1000), (2, 5000)])
def test_quantize_and_restore_bit_for_bit(rows, cols, fmt, dtype):
    x = rand(gen(rows + cols), rows, cols, spread=3.0, dtype=DT[dtype])
    q = block8.quantize(x, fmt)
    codes, e = R.split(x, fmt)
    assert same(q.codes.float().double(), codes)
    assert torch.equal(q.scales.view(torch.uint8).int(), (e + 127).int())
    pad = torch.as_strided(q.codes.view(torch.uint8), (rows, (cols + 15) // 16 * 16), (q.codes.stride(0), 1))[:, cols:]
    assert not bool(pad.any())
    for out in DT.values():
        assert same(block8.dequantize(q, out), R.values(x, fmt).to(torch.float32).to(out))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows, cols", [(3, 70001), (1, 300000), (17, 20000)])
def test_few_long_rows(rows, cols, dtype):
    """Rows that several workgroups share, as they are and as columns of a transposed matrix."""
    x = rand(gen(rows), rows, cols, spread=2.0, dtype=DT[dtype])
    codes, e = R.split(x, "e4m3")
    for y in (x, x.t().contiguous().t()):
        q = block8.quantize(y)
        assert same(q.codes.float().double(), codes) and torch.equal(q.scales.view(torch.uint8).int(), (e + 127).int())
        assert same(block8.dequantize(q, DT[dtype]), R.of(q).to(DT[dtype]))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows, cols", [(1, 130), (7, 9), (8, 128), (63, 129), (65, 127), (129, 200), (200, 1)])
def test_quantize_transposed(rows, cols, dtype):
    """Columns contiguous, columns an odd distance apart, an odd start: values behind the last row and column are NaN."""
    g = gen(rows + cols)
    for start, apart in ((0, rows + rows % 2), (1, rows + 3), (5, rows + 8)):
        store = torch.full((start + cols * apart + 300,), math.nan, dtype=DT[dtype], device="cuda")
        x = torch.as_strided(store, (rows, cols), (1, apart), start)
        x.copy_(rand(g, rows, cols, spread=2.0, dtype=DT[dtype]))
        for fmt in ("e4m3", "e5m2"):
            q = block8.quantize(x, fmt)
            codes, e = R.split(x.contiguous(), fmt)
            assert same(q.codes.float().double(), codes) and torch.equal(q.scales.view(torch.uint8).int(), (e + 127).int()), (start, apart, fmt)


@pytest.mark.parametrize("dtype", list(DT))
def test_quantize_strides(dtype):
    base = rand(gen(3), 300, 417, spread=2.0, dtype=DT[dtype])
    views = {"transposed": base.t(), "columns 1..": base[:, 1:], "every second row": base[::2], "every second column": base[:, ::2],
             "a transposed slice": base[5:70, 3:200].t(), "one row of a transposed view": base[:, :1].t(), "one column": base[:, 5:6],
             "expanded rows": base[:1].expand(9, 417), "expanded columns": base[:, :1].expand(300, 200), "a transposed row": base[:1].t(),
             "odd start": base.reshape(-1)[1:1 + 64 * 128].view(64, 128)}
    for name, x in views.items():
        for fmt in ("e4m3", "e5m2"):
            q = block8.quantize(x, fmt)
            codes, e = R.split(x, fmt)
            assert same(q.codes.float().double(), codes) and torch.equal(q.scales.view(torch.uint8).int(), (e + 127).int()), (name, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_edge_values(fmt):
    tiny, most = 2.0 ** -149, torch.finfo(torch.float32).max
    x = torch.zeros(10, 200)
    x[1, :3] = torch.tensor([tiny, -5 * tiny, 3e-40])
    x[2, :4] = torch.tensor([most, -most, 1.0, 1e30])
    x[3, 7] = math.nan
    x[3, 8:10] = torch.tensor([2.5, -1e-3])
    x[4, 3:6] = torch.tensor([math.inf, -math.inf, 7.0])
    x[5] = math.nan
    x[6, 130] = math.inf
    x[7] = -0.0
    x[8, :4] = torch.tensor([448.0, 448.0 * (1 + 2.0 ** -23), 57344.0, 1.75])
    x[9, :3] = torch.tensor([1.0, 2.0 ** -9, 2.0 ** -17 * 1.5])
    for y in (x.cuda(), x.cuda().t().contiguous().t()):
        q = block8.quantize(y, fmt)
        codes, e = R.split(y, fmt)
        assert torch.equal(q.scales.view(torch.uint8).int(), (e + 127).int())
        assert same(q.codes.float().double(), codes)
        assert same(block8.dequantize(q), R.values(y, fmt).float())


def test_dequantize_every_code_and_scale():
    """All codes of both formats under all 256 scale bytes (0 is 2^-127, 255 is NaN)."""
    for dt in (torch.float8_e4m3fn, torch.float8_e5m2):
        codes = torch.arange(256, dtype=torch.uint8).view(1, 256).repeat(256, 1).cuda().view(dt)
        scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 2).cuda().view(torch.float8_e8m0fnu)
        got = block8.dequantize(block8.Block8(codes, scales))
        s = torch.pow(2.0, torch.arange(256, dtype=torch.float64) - 127)
        s[255] = math.nan
        want = (codes.float().cpu().double() * s[:, None]).float()
        assert same(got.cpu(), want)


def test_rows_of_none():
    q = block8.quantize(torch.empty(0, 77, device="cuda"))
    assert q.shape == (0, 77) and block8.dequantize(q).shape == (0, 77)
    w = block8.quantize(rand(gen(), 5, 77))
    assert block8.matmul(q, w).shape == (0, 5) and block8.linear(torch.empty(2, 0, 77, device="cuda"), w).shape == (2, 0, 5)
    dw, db = block8.weight_grad(torch.empty(0, 5, device="cuda"), q, bias_dtype=torch.float32)
    assert dw.shape == (5, 77) and not bool(dw.any()) and db.shape == (5,) and not bool(db.any())


# ------------------------------------------------------------------------------------------------ products
SIZES = [(1, 1, 1), (1, 16, 128), (1, 4096, 512), (2, 3, 640), (5, 70, 31), (13, 200, 1000), (16, 64, 129), (17, 33, 255), (64, 64, 64), (100, 300, 513),
         (130, 257, 1000), (256, 256, 256), (300, 512, 1536), (700, 520, 2048), (31, 9, 9000)]


@pytest.mark.parametrize("M, N, K", SIZES)
@pytest.mark.parametrize("dtype", list(DT))
def test_matmul(M, N, K, dtype):
    g = gen(M * 7 + N + K)
    fa, fb = [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")][(M + N + K) % 4]
    a, b = block8.quantize(rand(g, M, K, spread=1.0), fa), block8.quantize(rand(g, N, K, spread=1.0), fb)
    bias = rand(g, N, dtype=DT[["f32", "bf16", "f16"][N % 3]]) if N % 2 else None
    va, vb = R.of(a), R.of(b)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    got = block8.matmul(a, b, bias, DT[dtype])
    close(got, ref, K + 1, mag, (M, N, K), True)
    # in the 2-norm: float32 sums, or the 8-bit instructions' loss and one rounding (at most eps / 2, taken three times over)
    off = float((got.double() - ref).norm() / ref.norm()) if bool(ref.any()) else 0.0
    assert off <= (1e-6 if dtype == "f32" else 1.5 * torch.finfo(DT[dtype]).eps) or M * N < 4, off


@pytest.mark.parametrize("fa", ["e4m3", "e5m2"])
@pytest.mark.parametrize("fb", ["e4m3", "e5m2"])
@pytest.mark.parametrize("M", [3, 200])
def test_matmul_formats_and_scales(M, fa, fb):
    """Whole numbers whose sums float32 holds exactly: the product is exact whatever the order, under very different scales."""
    g = gen(5)
    N, K = 90, 700
    a = torch.randint(-3, 4, (M, K), generator=g).float() * torch.pow(2.0, torch.randint(-3, 4, (M, 1), generator=g).float())
    b = torch.randint(-3, 4, (N, K), generator=g).float() * torch.pow(2.0, torch.randint(-3, 4, (N, 1), generator=g).float())
    for k in range(0, K, 128):
        b[:, k:k + 128] *= 2.0 ** (k // 128 % 3)
    a, b = a.cuda(), b.cuda()
    qa, qb = block8.quantize(a, fa), block8.quantize(b, fb)
    assert torch.equal(R.of(qa), a.double()) and torch.equal(R.of(qb), b.double())
    assert torch.equal(block8.matmul(qa, qb, dtype=torch.float32).double(), a.double() @ b.double().t())


def test_matmul_own_codes_and_odd_layouts():
    """Codes in contiguous rows of odd length, in a slice of a larger matrix with other codes around, and scales in wide rows."""
    g = gen(6)
    x, w = rand(g, 20, 150, spread=1.0), rand(g, 40, 150, spread=1.0)
    q, p = block8.quantize(x), block8.quantize(w)
    want = block8.matmul(q, p, dtype=torch.float32)
    tight = block8.Block8(q.codes.contiguous(), q.scales.contiguous())
    assert torch.equal(block8.matmul(tight, p, dtype=torch.float32), want)
    wide = torch.full((20, 256), 0x7F, dtype=torch.uint8, device="cuda")
    wide[:, 32:182] = q.codes.view(torch.uint8)
    assert torch.equal(block8.matmul(block8.Block8(wide.view(q.codes.dtype)[:, 32:182], q.scales), p, dtype=torch.float32), want)
    assert torch.equal(block8.matmul(q, block8.Block8(p.codes[::1], p.scales.contiguous()), dtype=torch.float32), want)
    one = block8.matmul(block8.Block8(q.codes[3:4], q.scales[3:4]), p, dtype=torch.float32)
    assert torch.allclose(one, want[3:4], rtol=1e-5, atol=1e-5)


def test_matmul_nan_and_infinity_stay_in_their_rows():
    g = gen(7)
    x, w = rand(g, 70, 300), rand(g, 50, 300)
    x[3, 200] = math.nan
    w[7, 5] = math.inf
    y = block8.matmul(block8.quantize(x), block8.quantize(w, "e5m2"), dtype=torch.float32)
    assert bool(y[3].isnan().all()) and not bool(y[:3, :7].isnan().any()) and not bool(y[4:, 8:].isnan().any())
    assert not bool(y[:, 7].isfinite().any())


@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (1, 5, 300), (7, 3, 64), (50, 64, 64), (64, 130, 96), (200, 64, 320), (333, 77, 129), (1000, 256, 512), (4097, 40, 200), (3000, 320, 130),
                                     (777, 2048, 1040), (65, 2056, 1030), (5000, 2048, 1024)])
@pytest.mark.parametrize("dtype", list(DT))
def test_weight_grad(M, N, K, dtype):
    g = gen(M + N + K)
    fmt = "e4m3" if (M + K) % 2 else "e5m2"
    q = block8.quantize(rand(g, M, K, spread=1.0), fmt)
    dy = rand(g, M, N, spread=1.0, dtype=DT[dtype])
    v = R.of(q)
    for out in (torch.float32, DT[dtype]):
        dw, db = block8.weight_grad(dy, q, out, out)
        # a float32 gradient is split in bf16 terms: their rest is below 2^-24 of it
        close(dw, dy.double().t() @ v, M + 1, dy.double().abs().t() @ v.abs(), (M, N, K))
        close(db, dy.double().sum(0), M, dy.double().abs().sum(0), (M, N, K))
    again, _ = block8.weight_grad(dy, q, torch.float32)
    assert torch.equal(again, block8.weight_grad(dy, q, torch.float32)[0])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M, N, K", [(71, 64, 64), (71, 2048, 1040), (71, 9, 64)])
def test_weight_grad_nan_and_infinity(M, N, K, dtype):
    """What is not finite in a gradient or in a checkpoint reaches its own row or column of dw, in the last rows too, and nothing else."""
    g = gen(40)
    q = block8.quantize(torch.ones(M, K).cuda() + torch.rand(M, K, generator=g).cuda())
    dy = rand(g, M, N, dtype=DT[dtype])
    dy[M - 1, 3], dy[M - 2, 5], dy[0, 7] = math.inf, math.nan, -math.inf
    dw, _ = block8.weight_grad(dy, q)
    assert bool((dw[3] == math.inf).all()) and bool(dw[5].isnan().all()) and bool((dw[7] == -math.inf).all())
    assert bool(dw[[i for i in range(N) if i not in (3, 5, 7)]].isfinite().all())
    x = torch.ones(M, K).cuda()
    x[M - 1, 6] = math.nan
    dw, _ = block8.weight_grad(rand(g, M, N, dtype=DT[dtype]), block8.quantize(x))
    assert bool(dw[:, 6].isnan().all()) and bool(dw[:, [i for i in range(K) if i != 6]].isfinite().all())


def test_weight_grad_is_exact_in_float32():
    """Gradients with 24 significant bits against codes 2^k: every product is exact, one term per sum."""
    g = gen(8)
    M = 96
    q = block8.quantize(torch.eye(M).cuda() * 2.0)
    dy = rand(g, M, 70, spread=5.0)
    assert torch.equal(block8.weight_grad(dy, q)[0], 2 * dy.t())


def test_weight_grad_strides_and_parts():
    g = gen(9)
    q = block8.quantize(rand(g, 120, 70))
    dy = rand(g, 120, 90)
    want = block8.weight_grad(dy, q, bias_dtype=torch.float32)
    wide = torch.full((120, 200), math.nan, device="cuda")
    wide[:, 33:123] = dy
    for x in (wide[:, 33:123], dy.t().contiguous().t()):
        got = block8.weight_grad(x, q, bias_dtype=torch.float32)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert block8.weight_grad(dy, q)[1] is None
    dw, db = block8.weight_grad(dy, q, bias_dtype=torch.float32, weight=False)
    assert dw is None and torch.equal(db, want[1])
    ones = torch.ones(1, 1, device="cuda").expand(120, 90)
    close(block8.weight_grad(ones, q)[0], ones.double().t() @ R.of(q), 121, ones.double().t() @ R.of(q).abs())


@pytest.mark.parametrize("M", [1, 2, 31, 32, 33, 63, 64, 65, 95, 96, 127, 129, 192, 1000])
@pytest.mark.parametrize("dtype", list(DT))
def test_weight_grad_row_counts(M, dtype):
    """Rows that fill the product's steps and rows that do not, with NaN behind the last one of both operands and beside the columns;
    and each of the two gradients alone."""
    g = gen(50 + M)
    N, K = 72, 136
    big = torch.full((M + 70, 96), math.nan, dtype=DT[dtype], device="cuda")
    big[:M, 16:16 + N] = rand(g, M, N, dtype=DT[dtype])
    dy = big[:M, 16:16 + N]
    x = torch.full((M + 70, K), math.nan, device="cuda")
    x[:M] = rand(g, M, K, spread=1.0)
    all_rows = block8.quantize(x)
    q = block8.Block8(all_rows.codes[:M], all_rows.scales[:M])
    v = R.of(q)
    dw, db = block8.weight_grad(dy, q, bias_dtype=torch.float32)
    close(dw, dy.double().t() @ v, M + 1, dy.double().abs().t() @ v.abs(), M)
    close(db, dy.double().sum(0), M, dy.double().abs().sum(0), M)
    assert torch.equal(block8.weight_grad(dy, q)[0], dw)
    assert torch.equal(block8.weight_grad(dy, q, bias_dtype=torch.float32, weight=False)[1], db)
    packed = dy.contiguous()                                                  # (rows 144 bytes apart instead of 192)
    assert torch.equal(block8.weight_grad(packed, q)[0], dw)


@pytest.mark.parametrize("dtype", list(DT))
def test_weight_grad_of_tiny_values(dtype):
    """Operands become bf16 terms, whose smallest step is 2^-133: a checkpoint's value, rounded to one, is off by at most half a step,
    a float32 gradient, cut off after its third, by less than a whole one."""
    g = gen(51)
    M, N, K = 200, 40, 70
    for sy, sx in ((-10 if dtype == "f16" else -120, 60), (5 if dtype == "f16" else 60, -128)):
        dy, q = (rand(g, M, N) * 2.0 ** sy).to(DT[dtype]), block8.quantize(rand(g, M, K) * 2.0 ** sx)
        v, d = R.of(q), dy.double()
        got = block8.weight_grad(dy, q)[0].double()
        mag = d.abs().t() @ v.abs()
        step = 2.0 ** -134 * d.abs().sum(0)[:, None] + 2.0 ** -133 * v.abs().sum(0)[None, :]
        assert bool(((got - d.t() @ v).abs() <= (M + 2) * 2.0 ** -23 * mag + step + 2.0 ** -149).all()), (sy, sx)


# ------------------------------------------------------------------------------------------------ the linear layer
@pytest.mark.parametrize("shape, N", [((1, 512), 256), ((3, 40), 7), ((2, 5, 200), 64), ((40, 1000), 130), ((300,), 20), ((260, 384), 300)])
@pytest.mark.parametrize("dtype", list(DT))
def test_linear(shape, N, dtype):
    g = gen(N)
    x, w = rand(g, *shape, spread=1.0, dtype=DT[dtype]), rand(g, N, shape[-1])
    wq = block8.quantize(w)
    bias = rand(g, N, dtype=DT[dtype])
    y = block8.linear(x, wq, bias)
    assert y.shape == shape[:-1] + (N,) and y.dtype == x.dtype
    v, u = R.values(x.reshape(-1, shape[-1])), R.of(wq)
    close(y.reshape(-1, N), v @ u.t() + bias.double(), shape[-1] + 1, v.abs() @ u.abs().t() + bias.double().abs(), "", True)


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 40])
def test_linear_is_quantize_and_matmul(rows):
    g = gen(rows)
    x, w = rand(g, rows, 1000, spread=1.0, dtype=torch.bfloat16), block8.quantize(rand(g, 333, 1000))
    assert torch.equal(block8.linear(x, w), block8.matmul(block8.quantize(x), w, dtype=torch.bfloat16))


@pytest.mark.parametrize("rows, K, N", [(16, 2048, 100), (16, 2049, 100), (1, 32768, 40), (1, 32769, 40), (5, 6553, 33), (3, 16, 1), (16, 8, 17)])
@pytest.mark.parametrize("dtype", list(DT))
def test_linear_of_few_rows(rows, K, N, dtype):
    """On both sides of the size up to which one launch does it all: the same result as quantizing and multiplying."""
    g = gen(rows + K)
    x, w, bias = rand(g, rows, K, spread=1.0, dtype=DT[dtype]), block8.quantize(rand(g, N, K)), rand(g, N)
    y = block8.linear(x, w, bias)
    assert same(y, block8.matmul(block8.quantize(x), w, bias, dtype=DT[dtype]))
    v, u = R.values(x), R.of(w)
    close(y, v @ u.t() + bias.double(), K + 1, v.abs() @ u.abs().t() + bias.double().abs(), (rows, K, N), product8=True)


@pytest.mark.parametrize("shape, N, bias", [((1, 64), 16, True), ((17, 33), 9, False), ((3, 50, 320), 64, True), ((300, 256), 200, True), ((1030, 130), 70, False)])
@pytest.mark.parametrize("dtype, wtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("grad_fmt", ["e4m3", "e5m2"])
def test_linear8_against_its_formula(shape, N, bias, dtype, wtype, grad_fmt):
    g = gen(N + len(shape))
    K = shape[-1]
    x, w = rand(g, *shape, spread=1.0, dtype=DT[dtype]).requires_grad_(), rand(g, N, K, dtype=DT[wtype]).requires_grad_()
    b = rand(g, N, dtype=DT[wtype]).requires_grad_() if bias else None
    y = train_ops.linear8(x, w, b, grad_fmt)
    gy = rand(g, *y.shape, spread=1.0, dtype=DT[dtype])
    y.backward(gy)
    qx, qw = R.values(x.detach().reshape(-1, K)), R.values(w.detach())
    g2 = gy.reshape(-1, N)
    qg, qwt = R.values(g2, grad_fmt), R.values(w.detach().t())
    M = g2.shape[0]
    off = b.detach().double() if bias else 0.0
    close(y.detach().reshape(-1, N), qx @ qw.t() + off, K + 1, qx.abs() @ qw.abs().t() + (off.abs() if bias else 0.0), "y", True)
    close(x.grad.reshape(-1, K), qg @ qwt.t(), N, qg.abs() @ qwt.abs().t(), "dx", True)
    close(w.grad, g2.double().t() @ qx, M + 1, g2.double().abs().t() @ qx.abs(), "dw")
    assert x.grad.dtype == x.dtype and w.grad.dtype == w.dtype
    if bias:
        close(b.grad, g2.double().sum(0), M, g2.double().abs().sum(0), "db")


def test_linear8_against_differences():
    """Values that 8 bits hold exactly, also after a step: the layer is linear there, so central differences are its gradient."""
    g = gen(11)
    M, N, K = 6, 20, 140
    ints = lambda *s: torch.randint(-6, 7, s, generator=g).float().cuda()      # noqa: E731
    x, w, gy = ints(M, K), ints(N, K), ints(M, N)
    x[:, 0] = x[:, 130] = w[:, 0] = w[:, 130] = 8.0                           # the blocks' largest: scales stay as they are
    b = ints(N)
    xl, wl, bl = (t.clone().requires_grad_() for t in (x, w, b))
    train_ops.linear8(xl, wl, bl).backward(gy)

    def loss(x, w, b):
        return float((train_ops.linear8(x, w, b).double() * gy.double()).sum())
    for t, grad, at in ((x, xl.grad, [(0, 1), (3, 77), (5, 139)]), (w, wl.grad, [(0, 5), (19, 131), (7, 60)]), (b, bl.grad, [(0,), (19,)])):
        for i in at:
            lo, hi = t.clone(), t.clone()
            lo[i] -= 1
            hi[i] += 1
            args = [(lo if u is t else u, hi if u is t else u) for u in (x, w, b)]
            d = (loss(*(a[1] for a in args)) - loss(*(a[0] for a in args))) / 2
            assert d == float(grad[i]), (i, d, float(grad[i]))


def test_linear8_parts_of_the_gradient():
    g = gen(12)
    x, w, b = rand(g, 30, 64), rand(g, 16, 64), rand(g, 16)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    gy = rand(g, 30, 16)
    train_ops.linear8(*full).backward(gy)
    for need in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        train_ops.linear8(*leaves).backward(gy)
        for i, t in enumerate(leaves):
            assert (t.grad is None) if not need >> i & 1 else torch.equal(t.grad, full[i].grad)
    y = train_ops.linear8(full[0], full[1])
    y.sum().backward()                                                       # an expanded gradient
    assert torch.isfinite(full[0].grad).all()
    with torch.no_grad():
        assert not train_ops.linear8(full[0], full[1]).requires_grad


def test_second_derivatives_are_refused():
    g = gen(15)
    x, w = rand(g, 8, 64).requires_grad_(), rand(g, 16, 64).requires_grad_()
    r, b, l = (t.requires_grad_() for t in (torch.nn.functional.pad(rand(g, 1, 4, 4, 64), (0, 0, 1, 1, 1, 1)), rand(g, 64), rand(g, 64)))
    for y, leaf in ((train_ops.linear8(x, w), x), (train_ops.an_relu8_ring(r, b, l)[0], r)):
        d, = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            d.sum().backward()


def test_rows_far_apart():
    """Rows of gradients and codes further apart than the products reach, and single rows with such a stride."""
    g = gen(16)
    far = (1 << 23) + 16
    store = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device="cuda")
    dy = torch.as_strided(store, (3, 64), (far, 1))
    dy.copy_(rand(g, 3, 64))
    q = block8.quantize(rand(g, 3, 40))
    assert torch.equal(block8.weight_grad(dy, q)[0], block8.weight_grad(dy.contiguous(), q)[0])
    assert torch.equal(block8.weight_grad(dy[:1], block8.Block8(q.codes[:1], q.scales[:1]))[0],
                       block8.weight_grad(dy[:1].contiguous(), block8.Block8(q.codes[:1].contiguous(), q.scales[:1]))[0])
    p = block8.quantize(dy)
    assert torch.equal(p.codes.float(), block8.quantize(dy.contiguous()).codes.float())
    codes = torch.as_strided(store.view(torch.uint8).view(p.codes.dtype), (3, 64), (far, 1))
    codes.view(torch.uint8).copy_(p.codes.view(torch.uint8))
    w = block8.quantize(rand(g, 50, 64))
    want = block8.matmul(p, w)
    assert torch.equal(block8.matmul(block8.Block8(codes, p.scales), w), want)
    assert torch.equal(block8.matmul(block8.Block8(codes[:1], p.scales[:1]), w), block8.matmul(block8.Block8(p.codes[:1], p.scales[:1]), w))
    assert torch.equal(block8.linear(torch.as_strided(store, (1, 64), (far, 1), 8), w), block8.linear(store[8:72], w)[None])


def test_linear8_refuses_a_changed_weight():
    g = gen(13)
    x, w = rand(g, 8, 64).requires_grad_(), rand(g, 16, 64).requires_grad_()
    y = train_ops.linear8(x, w)
    with torch.no_grad():
        w += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_refusals():
    g = gen(14)
    x, w = rand(g, 4, 64), block8.quantize(rand(g, 8, 64))
    with pytest.raises(ValueError):
        block8.quantize(x, "e3m4")
    with pytest.raises(TypeError):
        block8.quantize(x.double())
    with pytest.raises(AssertionError):
        block8.quantize(x[0])
    with pytest.raises(AssertionError):
        block8.quantize(x[:, :0])
    with pytest.raises(TypeError):
        block8.dequantize(w, torch.float64)
    with pytest.raises(AssertionError):
        block8.matmul(block8.quantize(x[:, :32]), w)
    with pytest.raises(TypeError):
        block8.matmul(x, w)
    with pytest.raises(AssertionError):
        block8.linear(x, w, torch.zeros(7, device="cuda"))
    with pytest.raises(hip.InterflowHipError):
        block8.linear(x, w, torch.zeros(8))
    with pytest.raises(AssertionError):
        block8.linear(x[:, :60], w)
    with pytest.raises(TypeError):
        block8.linear(x, x)
    with pytest.raises(TypeError):
        block8.Block8(x, w.scales)
    with pytest.raises(AssertionError):
        block8.Block8(w.codes, w.scales[:4])
    with pytest.raises(AssertionError):
        block8.weight_grad(x[:3], block8.quantize(x))
    with pytest.raises(ValueError):
        train_ops.linear8(x, x, grad_fmt="bf16")
    with pytest.raises(AssertionError):
        train_ops.linear8(x, x[:, :60])
    r = torch.zeros(1, 6, 6, 48, device="cuda")
    with pytest.raises(NotImplementedError):
        train_ops.an_relu8_ring(r, torch.zeros(48, device="cuda"), torch.zeros(48, device="cuda"))
    r = torch.zeros(1, 6, 6, 64, device="cuda")
    with pytest.raises(AssertionError):
        train_ops.an_relu8_ring(r, torch.zeros(32, device="cuda"), torch.zeros(64, device="cuda"))
    with pytest.raises(TypeError):
        train_ops.an_relu8_ring(r.half(), torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda"))


# ------------------------------------------------------------------------------------------------ ActNorm + ReLU
def ring(x):
    return torch.nn.functional.pad(x, (0, 0, 1, 1, 1, 1))


@pytest.mark.parametrize("B, h, w, C", [(1, 1, 1, 32), (1, 3, 5, 64), (2, 10, 10, 64), (3, 7, 9, 96), (1, 16, 33, 128), (2, 5, 4, 320), (1, 2, 3, 1024), (4, 40, 40, 64), (1, 60, 300, 32)])
def test_an_relu8(B, h, w, C):
    g = gen(B + h + w + C)
    x = ring(rand(g, B, h, w, C, spread=2.0))
    x[:, 0] = math.nan                                                        # ring pixels are not read
    gy = ring(rand(g, B, h, w, C))
    gy[:, :, 0] = math.nan
    bias, logs = rand(g, 1, C, 1, 1), 0.5 * rand(g, 1, C, 1, 1)
    xl, bl, ll = (t.clone().requires_grad_() for t in (x, bias, logs))
    y, ck = train_ops.an_relu8_ring(xl, bl, ll)
    y.backward(gy)
    xi, gi = x[:, 1:-1, 1:-1], gy[:, 1:-1, 1:-1].double()
    s = logs.double().exp().view(-1)
    v = (xi + bias.view(-1)).relu()                                           # one float32 addition: what the checkpoint holds
    q = R.values(v.reshape(-1, C), keep_positive=True).view(v.shape)
    codes = ring(R.split(v.reshape(-1, C), "e4m3", keep_positive=True)[0].view(v.shape))
    assert torch.equal(ck.codes.float().double(), codes)
    # y and dx: one product with exp(logs), which is off by a few units of its last place
    eps = 2.0 ** -21
    ref = ring((xi.double() + bias.double().view(-1)).relu() * s)
    assert bool(((y.double() - ref).abs() <= eps * ref.abs() + 2.0 ** -23 * ring((xi.double().abs() + bias.double().view(-1).abs()) * s)).all())
    ref = ring(gi * (v > 0) * s)
    assert bool(((xl.grad.double() - ref).abs() <= eps * ref.abs()).all())
    n = B * h * w
    m = gi.abs() * (v > 0)
    assert bl.grad.shape == bias.shape and ll.grad.shape == logs.shape
    for got, ref, mag in ((bl.grad, (gi * (v > 0)).sum((0, 1, 2)), m.sum((0, 1, 2))), (ll.grad, (gi * q).sum((0, 1, 2)), (gi.abs() * q).sum((0, 1, 2)))):
        assert bool(((got.view(-1).double() - ref * s).abs() <= (n * 2.0 ** -23 + 2.0 ** -20) * mag * s).all())
    back = ck.restore().double()
    ref = ring(q * s)
    assert bool(((back - ref).abs() <= eps * ref.abs()).all())


def test_an_relu8_matches_the_float32_operator():
    """y and dx are those of an_relu_ring, bit for bit; its own gradients on values that 8 bits hold exactly are too."""
    g = gen(21)
    x = ring(torch.randint(-8, 9, (2, 9, 11, 64), generator=g).float().cuda())
    gy = ring(torch.randint(-4, 5, (2, 9, 11, 64), generator=g).float().cuda())
    bias, logs = torch.randint(-2, 3, (64,), generator=g).float().cuda(), torch.zeros(64, device="cuda")
    out = []
    for f in (train_ops.an_relu_ring, lambda *a: train_ops.an_relu8_ring(*a)[0]):
        l = [t.clone().requires_grad_() for t in (x, bias, logs)]
        y = f(*l)
        y.backward(gy)
        out.append([y.detach()] + [t.grad for t in l])
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_an_relu8_against_differences():
    """bias by central differences of the float32 operator; logs by those of the function the checkpoint stands for: its values
    (all of x + bias but 8.5, which has five significant bits and is kept as 8) times exp(logs)."""
    g = gen(22)
    x = ring(torch.randint(-8, 9, (1, 6, 7, 32), generator=g).float().cuda()) + 0.0
    gy = ring(rand(g, 1, 6, 7, 32))
    bias, logs = torch.full((32,), 0.5).cuda(), 0.2 * rand(g, 32)              # x + bias: never 0
    bl, ll = bias.clone().requires_grad_(), logs.clone().requires_grad_()
    train_ops.an_relu8_ring(x, bl, ll)[0].backward(gy)
    xi, gi = x[:, 1:-1, 1:-1], gy[:, 1:-1, 1:-1].double()
    kept = R.values((xi + bias).relu().reshape(-1, 32), keep_positive=True).view(xi.shape)
    assert torch.equal(kept != (xi + bias).relu(), xi == 8)

    def loss(b, l):
        return ((xi.double() + b).relu() * l.exp() * gi).sum((0, 1, 2))
    d = 1e-3
    db = (loss(bias.double() + d, logs.double()) - loss(bias.double() - d, logs.double())) / (2 * d)
    dl = ((kept * (logs.double() + d).exp() * gi).sum((0, 1, 2)) - (kept * (logs.double() - d).exp() * gi).sum((0, 1, 2))) / (2 * d)
    mag = loss(bias.double(), logs.double()).abs().max() + 20
    assert float((bl.grad.double() - db).abs().max()) <= 1e-5 * float(mag)
    assert float((ll.grad.double() - dl).abs().max()) <= (d * d / 6 + 1e-5) * float(mag) * 10


@pytest.mark.parametrize("k, cin, cout", [(1, 64, 64), (3, 64, 24), (1, 128, 96)])
def test_convolution_from_a_checkpoint(k, cin, cout):
    """The weight gradient behind a checkpoint is the convolution's own on the restored activation; y, dx and dbias do not change."""
    g = gen(k + cin)
    x, bias, logs = ring(rand(g, 2, 9, 8, cin)), rand(g, cin), 0.3 * rand(g, cin)
    w, b = rand(g, cout, cin, k, k), rand(g, cout)
    gy = torch.nn.functional.pad(rand(g, 2, 9, 8, cout), (0, train_ops.pad32(cout) - cout, 1, 1, 1, 1))

    def step(mode):
        l = [t.clone().requires_grad_() for t in (x, bias, logs, w, b)]
        a, ck = train_ops.an_relu8_ring(*l[:3])
        if mode == "restored":
            a = a + (ck.restore() - a).detach()                               # the value is the restored one
            ck = None
        y = train_ops.conv2d_ring([a], [cin], l[3], l[4], [ck] if mode == "8 bit" else None)
        y.backward(gy)
        return [y.detach()] + [t.grad for t in l]
    plain, kept, restored = step("plain"), step("8 bit"), step("restored")
    for i in (0, 1, 2, 3, 5):
        assert torch.allclose(kept[i], plain[i], rtol=1e-6, atol=1e-6 * float(plain[i].abs().max())), i
    n = 2 * 9 * 8
    assert float((kept[4] - restored[4]).abs().max()) <= 4 * n * 2.0 ** -23 * float(x.abs().max() * 4) * float(gy.abs().max()) * n
    rel = float((kept[4] - plain[4]).norm() / plain[4].norm())
    assert 0 < rel < 2.0 ** -4, rel


def test_a_checkpoints_logs_may_not_change_before_they_are_used():
    g = gen(23)
    x, bias, logs = ring(rand(g, 1, 4, 5, 64)), rand(g, 64), 0.3 * rand(g, 64)
    _, used = train_ops.an_relu8_ring(x, bias, logs)
    want = used.restore()
    _, late = train_ops.an_relu8_ring(x, bias, logs)
    logs += 1
    assert torch.equal(used.restore(), want)
    with pytest.raises(RuntimeError):
        late.restore()


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
BIG = (70001, 32768)                                                          # 2.3e9 values; the last rows lie behind 2^31


def _big(dtype):
    return torch.randn(BIG, generator=torch.Generator("cuda").manual_seed(60), device="cuda", dtype=dtype)


def test_large_quantize_restore_and_products():
    x = _big(torch.bfloat16)
    q = block8.quantize(x)
    tail, rows = x[-3:].clone(), slice(BIG[0] - 3, BIG[0])
    want = block8.quantize(tail)
    assert torch.equal(q.codes[rows].float(), want.codes.float()) and torch.equal(q.scales[rows].float(), want.scales.float())
    assert torch.equal(block8.dequantize(q, torch.bfloat16)[rows], block8.dequantize(want, torch.bfloat16))
    t = block8.quantize(x.t())                                                # its last block of columns: x's last rows
    assert torch.equal(t.codes[-70:, -1].float(), block8.quantize(x[-(BIG[0] % 128):, -70:].t()).codes[:, -1].float())
    del t
    g = gen(61)
    w = block8.quantize(rand(g, 64, BIG[1]))
    v, u = R.of(want), R.of(w)
    close(block8.matmul(q, w, dtype=torch.float32)[rows], v @ u.t(), BIG[1], v.abs() @ u.abs().t())
    close(block8.linear(x, w)[rows], v @ u.t(), BIG[1], v.abs() @ u.abs().t(), product8=True)
    dy = rand(g, BIG[0], 8, dtype=torch.bfloat16)
    dw = block8.weight_grad(dy, q)[0][:, -5:]
    cols = block8.dequantize(q, torch.bfloat16)[:, -5:].double()
    close(dw, dy.double().t() @ cols, BIG[0], dy.double().abs().t() @ cols.abs())


def test_large_results_and_gradients():
    g = gen(62)
    a, b = block8.quantize(rand(g, BIG[0], 128)), block8.quantize(rand(g, BIG[1], 128))
    y = block8.matmul(a, b)
    v, u = R.of(block8.Block8(a.codes[-3:], a.scales[-3:])), R.of(b)
    close(y[-3:], v @ u.t(), 128, v.abs() @ u.abs().t(), product8=True)
    del y
    dy, q = _big(torch.float32), block8.quantize(rand(g, BIG[0], 8))
    dw, db = block8.weight_grad(dy, q, bias_dtype=torch.float32)
    cols, v = dy[:, -5:].double(), R.of(q)
    close(dw[-5:], cols.t() @ v, BIG[0] + 1, cols.abs().t() @ v.abs())
    close(db[-5:], cols.sum(0), BIG[0], cols.abs().sum(0))


def test_large_an_relu8():
    x = torch.randn(1, 1500, 1500, 1024, generator=torch.Generator("cuda").manual_seed(63), device="cuda")
    bias, logs = rand(gen(64), 1024), 0.1 * rand(gen(65), 1024)
    leaf = x.detach().requires_grad_()
    y, ck = train_ops.an_relu8_ring(leaf, bias, logs)
    small = x[:, -3:, -4:].contiguous()                                      # the last two inner pixels of the last inner row
    ys, cs = train_ops.an_relu8_ring(small, bias, logs)
    assert torch.equal(y[:, -2, -3:], ys[:, -2, -3:])
    assert torch.equal(ck.codes[:, -2, -3:].float(), cs.codes[:, -2, -3:].float())
    y.backward(x)
    want = torch.where(ys[:, -2, -3:-1] > 0, small[:, -2, -3:-1] * logs.exp(), 0.0)
    assert torch.allclose(leaf.grad[:, -2, -3:-1], want, rtol=2.0 ** -21, atol=0)


# ------------------------------------------------------------------------------------------------ streams, graphs, two at once
def test_on_another_stream_and_concurrently():
    g = gen(31)
    x, w, gy = rand(g, 300, 512, dtype=torch.bfloat16), rand(g, 256, 512, dtype=torch.bfloat16), rand(g, 300, 256, dtype=torch.bfloat16)

    def step():
        l = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        y = train_ops.linear8(*l)
        y.backward(gy)
        return [y.detach(), l[0].grad, l[1].grad]
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 13, 300])
def test_captured_and_replayed(rows):
    """linear and quantize / dequantize in a graph: replays on new inputs, with eager work in between."""
    g = gen(32)
    w = block8.quantize(rand(g, 200, 640))
    x = rand(g, rows, 640, dtype=torch.bfloat16)
    fn = lambda: (block8.linear(x, w), block8.dequantize(block8.quantize(x, "e5m2"), torch.bfloat16))      # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    for i in range(4):
        x.copy_(rand(g, rows, 640, dtype=torch.bfloat16))
        graph.replay()
        want = fn()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i


def test_training_step_captured_and_replayed():
    g = gen(33)
    x, w, b, gy = rand(g, 200, 320), rand(g, 64, 320), rand(g, 64), rand(g, 200, 64)
    r, rb, rl, rg = ring(rand(g, 2, 10, 12, 64)), rand(g, 64), 0.2 * rand(g, 64), ring(rand(g, 2, 10, 12, 64))

    def step():
        l = [t.detach().requires_grad_() for t in (x, w, b)]
        a = [t.detach().requires_grad_() for t in (r, rb, rl)]
        y = train_ops.linear8(*l)
        z, ck = train_ops.an_relu8_ring(*a)
        return [y.detach(), z.detach(), *torch.autograd.grad(y, l, gy), *torch.autograd.grad(z, a, rg), ck.restore()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(rand(g, 200, 320))
        r.copy_(ring(rand(g, 2, 10, 12, 64)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c), i


# ------------------------------------------------------------------------------------------------ the training path
def _flow(seed=0):
    from interflow_amd import synth
    from interflow_amd.flow_model import InterpFlow
    model = InterpFlow([2, 4])
    model.load_state_dict({k: torch.from_numpy(v) for k, v in synth.synth_interpflow_state([2, 4], seed=seed).items()}, strict=True)
    return model.cuda().train()


def test_training_path_with_8bit_checkpoints():
    """The flow's gradient-enabled passes: outputs and the gradient towards the input are the float32 path's, gradients behind a
    checkpoint are within the format's error, and less memory is held between forward and backward."""
    from interflow_amd import synth
    B, H = 2, 32
    x = torch.from_numpy(synth.synth_images(5, B, H, H)).cuda()
    feats = {k: torch.from_numpy(v).cuda() for k, v in synth.synth_features(6, B, H, H).items()}
    res = {}
    fused, train_flow.FUSED_LEVELS = train_flow.FUSED_LEVELS, False
    try:
        for bits in (32, 8):
            prev = train_flow.set_activation_checkpoints(bits)
            try:
                model = _flow()
                torch.cuda.synchronize()
                before = torch.cuda.memory_allocated()
                xi = x.clone().requires_grad_()
                z, ld = model(xi, None, lr_enc=feats, add_gt_noise=False, calc_loss=False)
                torch.cuda.synchronize()
                held = torch.cuda.memory_allocated() - before
                ((z ** 2).mean() - 1e-4 * ld.mean()).backward()
                res[bits] = (z.detach(), ld.detach(), xi.grad, {n: p.grad.clone() for n, p in model.flow_upsampler.named_parameters() if p.grad is not None}, held)
            finally:
                train_flow.set_activation_checkpoints(prev)
    finally:
        train_flow.FUSED_LEVELS = fused
    a, b = res[32], res[8]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert float((a[2] - b[2]).norm()) <= 1e-4 * float(a[2].norm())
    assert a[3].keys() == b[3].keys() and len(a[3]) > 500
    worst = 0.0
    for n in a[3]:
        if float(a[3][n].norm()) > 0:
            worst = max(worst, float((a[3][n] - b[3][n]).norm() / a[3][n].norm()))
    # an activation is off by at most 2^-4 of itself; a gradient is a sum over them, whose terms partly cancel
    print("largest relative difference of a gradient", worst, "held", a[4], b[4])
    assert 0 < worst < 0.25
    assert b[4] < 0.75 * a[4]
