"""Weight gradients from 8-bit checkpoints: what is not finite, and every kernel that a size may go to."""
import math

import pytest
import torch

from interflow_amd import block8
from tests import _block8_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M, N, K", [(71, 64, 64), (71, 2048, 1040), (130, 9, 200)])
def test_infinities_of_a_checkpoint(M, N, K, dtype):
    """An infinity times a gradient is an infinity of its sign, times zero or NaN it is NaN; every other column is as without it."""
    g = gen(M + N)
    x = torch.randn(M, K, generator=g)
    x[M - 1, 6] = math.inf
    dy = torch.randn(M, N, generator=g)
    dy[M - 1, :8] = torch.tensor([1.0, -1.0, 1.5, -0.0078125, math.inf, -math.inf, 0.0, math.nan])
    dy[M - 1, 8] = 1 + 2.0 ** -9                                             # (a second term of one bit)
    dy = dy.to(DT[dtype]).cuda()
    q = block8.quantize(x.cuda(), "e5m2")
    dw, _ = block8.weight_grad(dy, q)
    last = dy[M - 1].float()
    want = torch.where(last == 0, math.nan, last * math.inf)
    assert torch.equal(dw[:, 6].isnan(), want.isnan()) and torch.equal(dw[:, 6].nan_to_num(0.0), want.nan_to_num(0.0))
    others = [k for k in range(K) if k != 6]
    rows = [n for n in range(N) if n not in (4, 5, 7)]
    v, d = R.of(q)[:, others], dy.double()[:, rows]
    err = (M + 1) * 2.0 ** -23 * (d.abs().t() @ v.abs())
    assert bool(((dw[rows][:, others].double() - d.t() @ v).abs() <= err).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_terms_of_a_gradient_are_exact_beside_infinities(dtype):
    """One product per sum, times 2: the gradient's terms join to all its bits, whatever they are."""
    M, g = 96, gen(3)
    q = block8.quantize(torch.eye(M).cuda() * 2.0, "e5m2")
    dy = torch.randn(M, 70, generator=g) * torch.exp(3 * torch.randn(M, 70, generator=g))
    bits = torch.randint(0, 24, (M, 70), generator=g)
    f, e = torch.frexp(dy)
    dy = torch.ldexp(torch.trunc(f * 2.0 ** bits.float()), e - bits).clamp(-32752, 32752)         # 0 to 23 significant bits, finite in float16 (infinity times the zeros of q is NaN)
    dy = dy.to(DT[dtype]).cuda()
    assert torch.equal(block8.weight_grad(dy, q)[0], 2 * dy.t().float())


@pytest.mark.parametrize("dtype", list(DT))
def test_whole_numbers_beside_infinities(dtype):
    """Sums that float32 holds stay exact under an e5m2 checkpoint: what makes its terms all non-zero is below what a sum keeps."""
    M, N, K, g = 700, 60, 90, gen(4)
    dy = torch.randint(-9, 10, (M, N), generator=g).to(DT[dtype]).cuda()
    x = torch.randint(-3, 4, (M, K), generator=g).float().cuda()
    assert torch.equal(block8.weight_grad(dy, block8.quantize(x, "e5m2"))[0].double(), dy.double().t() @ x.double())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("M", [2, 7, 33])
def test_sums_that_cancel_are_zero(M, fmt, dtype):
    g = gen(M)
    dy = torch.randint(-2, 3, (M, 60), generator=g).to(DT[dtype]).cuda()
    x = torch.randint(-2, 3, (M, 90), generator=g).float().cuda()
    ref = dy.double().t() @ x.double()
    assert int(((ref == 0) & ((dy != 0).double().t() @ (x != 0).double() > 0)).sum()) > 100
    assert torch.equal(block8.weight_grad(dy, block8.quantize(x, fmt))[0].double(), ref)
