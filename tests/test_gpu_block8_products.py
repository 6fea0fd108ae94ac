"""Products of 8-bit blocks keep 24 bits, in every kernel that a size may go to."""
import pytest
import torch

from interflow_amd import block8, train_ops
from tests import _block8_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cancelling(g, rows, other, K):
    """a [rows, K] and b [other, K] that 8 bits hold exactly: every 8 neighbours of a row of a are 256, -256 and six of at most 3/64,
    which meet equal values of b.  The products of the first two cancel; with them in a sum of fewer than 17 bits the others are
    lost.  All partial sums, in any order, are multiples of 1/64 below 2^17 at these K: float32 holds them exactly."""
    a = torch.randint(-3, 4, (rows, K // 8, 8), generator=g).float() / 64
    a[:, :, 0] = 256.0
    a[:, :, 1] = -256.0
    b = torch.randint(1, 3, (other, K // 8, 1), generator=g).float() * (torch.randint(0, 2, (other, K // 8, 1), generator=g) * 2 - 1)
    return a.view(rows, K).cuda(), b.expand(other, K // 8, 8).reshape(other, K).cuda()


# few rows (one fragment, two), 64 x 64 with K split and whole, 128 x 128, 256 x 256
SIZES = [(1, 40, 1024), (16, 40, 4096), (20, 40, 1024), (40, 50, 2048), (200, 1000, 1032), (1500, 2000, 264), (2000, 2040, 520), (3500, 3600, 520)]


@pytest.mark.parametrize("M, N, K", SIZES)
@pytest.mark.parametrize("dtype", list(DT))
def test_products_keep_what_cancellation_leaves(M, N, K, dtype):
    a, b = cancelling(gen(M + N + K), M, N, K)
    ref = (a.double() @ b.double().t()).to(DT[dtype])
    assert float(ref.abs().max()) > 1
    for fa, fb in (("e4m3", "e4m3"), ("e4m3", "e5m2")):
        p, q = block8.quantize(a, fa), block8.quantize(b, fb)
        assert torch.equal(R.of(p), a.double()) and torch.equal(R.of(q), b.double())
        assert torch.equal(block8.matmul(p, q, dtype=DT[dtype]), ref)
    w = block8.quantize(b)
    assert torch.equal(block8.linear(a.to(DT[dtype]), w), ref)


@pytest.mark.parametrize("M, N, K", [(12, 512, 40), (40, 1024, 64), (300, 264, 1000)])
@pytest.mark.parametrize("dtype", list(DT))
def test_layer_keeps_what_cancellation_leaves(M, N, K, dtype):
    """y sums over K, dx over N."""
    g = gen(M + N)
    a, b = cancelling(g, M, N, K)
    w = b.clone().requires_grad_()
    y = train_ops.linear8(a.to(DT[dtype]), w)
    assert torch.equal(y, (a.double() @ b.double().t()).to(DT[dtype]))
    gy, wt = cancelling(g, M, K, N)
    x = torch.zeros(M, K, dtype=DT[dtype], device="cuda", requires_grad=True)
    train_ops.linear8(x, wt.t()).backward(gy.to(DT[dtype]))
    assert torch.equal(x.grad, (gy.double() @ wt.double().t()).to(DT[dtype]))


@pytest.mark.parametrize("M, N, K", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_8bit_instructions_on_request(M, N, K, dtype):
    """exact=False: off by at most 7 2^-13 of the products' magnitudes, and by one rounding; float32 results are the exact ones."""
    g = gen(M + K)
    a, b = block8.quantize(torch.randn(M, K, generator=g).cuda()), block8.quantize(torch.randn(N, K, generator=g).cuda())
    va, vb = R.of(a), R.of(b)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    err = (7 * 2.0 ** -13 + K * 2.0 ** -23) * mag
    tol = err + torch.finfo(DT[dtype]).eps / 2 * (ref.abs() + err) + torch.finfo(DT[dtype]).tiny
    y = block8.matmul(a, b, dtype=DT[dtype], exact=False)
    assert bool(((y.double() - ref).abs() <= tol).all())
    assert torch.equal(block8.matmul(a, b, dtype=torch.float32, exact=False), block8.matmul(a, b, dtype=torch.float32))
    x = va.to(DT[dtype])
    qx = R.values(x)
    ref, mag = qx @ vb.t(), qx.abs() @ vb.abs().t()
    err = (7 * 2.0 ** -13 + K * 2.0 ** -23) * mag
    tol = err + torch.finfo(DT[dtype]).eps / 2 * (ref.abs() + err) + torch.finfo(DT[dtype]).tiny
    assert bool(((block8.linear(x, b, exact=False).double() - ref).abs() <= tol).all())
    y = train_ops.linear8(x, vb.float(), exact=False)
    assert bool(((y.double() - qx @ R.values(vb).t()).abs() <= tol).all())


@pytest.mark.parametrize("M", [5, 100, 2040])
@pytest.mark.parametrize("ea, eb", [(-110, 60), (100, -126), (-60, -60), (60, 60), (-126, 126)])
def test_products_of_far_scales(M, ea, eb):
    """Whole numbers times powers of two near the ends of the range: exact as long as float32 has every partial sum, that is where the
    products' magnitudes add up to less than 2^128 (at 2^60 times 2^60: to less than 256)."""
    g = gen(M)
    K = 264 if M < 2000 else 1500
    a, b = torch.randint(-3, 4, (M, K), generator=g).float().cuda(), torch.randint(-3, 4, (M, K), generator=g).float().cuda()
    p, q = block8.quantize(a * 2.0 ** ea), block8.quantize(b * 2.0 ** eb)
    assert torch.equal(R.of(p), a.double() * 2.0 ** ea)
    ref = (a.double() @ b.double().t()) * 2.0 ** (ea + eb)
    held = (a.double().abs() @ b.double().abs().t()) * 2.0 ** (ea + eb) < 2.0 ** 128
    got = block8.matmul(p, q, dtype=torch.float32).double()
    assert torch.equal(torch.where(held, got, 0.0), torch.where(held, ref, 0.0)) and (bool(held.all()) or ea + eb == 120)
