"""The kernels of large products and weight gradients: whole results, on operands whose sums float32 holds exactly in any order (so do the
8-bit instructions: no product is below 2^-13 of another one in its block).  The plan is asked for, so that a size whose kernel
changes with the rules is noticed here."""
import pytest
import torch

from interflow_amd import block8, hip, train_ops
from tests import _block8_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPE = {"f32": 0, "bf16": 1, "f16": 2}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def ints(g, rows, cols, most):
    return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda").float()


def scaled(g, rows, cols, most=3):
    """Whole numbers times a power of two per row and one per block of 128: other scales from row to row and from step to step."""
    x = ints(g, rows, cols, most) * torch.pow(2.0, torch.randint(-2, 3, (rows, 1), generator=g, device="cuda").float())
    for k in range(0, cols, 128):
        x[:, k:k + 128] *= 2.0 ** (k // 128 * 5 % 3)
    return x


# M, N, K, tile: whole steps of 128 alone and with a rest, one step and less, odd and even numbers of them, remainders of the tile on both sides
PRODUCTS = [(8200, 4100, 100, 256), (8195, 4099, 128, 256), (3500, 3511, 300, 256), (3500, 3511, 640, 256), (3500, 3511, 1100, 256), (3333, 3600, 1024, 256),
            (2040, 2047, 1500, 128), (2047, 2033, 1536, 128), (1960, 2040, 1664, 128), (1000, 1030, 1030, 64), (500, 520, 2000, 64)]


@pytest.mark.parametrize("dtype, exact", [("f32", True), ("bf16", True), ("bf16", False), ("f16", True), ("f16", False)])
@pytest.mark.parametrize("M, N, K, tile", PRODUCTS)
def test_products(M, N, K, tile, dtype, exact):
    assert hip.lib().ifl_block8_matmul_plan(M, N, K) & 0xffff == tile
    g = gen(M + K)
    a, b = scaled(g, M, K), scaled(g, N, K)
    assert 9 * 16 * K < 1 << 24                                              # (of a row's and a column's own units)
    bias = ints(g, 1, N, 8)[0].to(DT[["f32", "bf16", "f16"][N % 3]]) if (M + N) % 2 else None
    fa, fb = [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")][PRODUCTS.index((M, N, K, tile)) % 4]
    qa, qb = block8.quantize(a, fa), block8.quantize(b, fb)
    ref = a.double() @ b.double().t()
    if bias is not None:
        ref += bias.double()
    assert torch.equal(ref.float().double(), ref)
    assert torch.equal(block8.matmul(qa, qb, bias, DT[dtype], exact=exact), ref.to(DT[dtype]))


# M, N, K, gradients' type, their first element's place, tile: rows that no step fills, parts of the sum, gradients read in place (bf16, whole aligned
# 16 bytes) and not
GRADIENTS = [(6200, 2048, 2040, "bf16", 0, 256), (6200, 2044, 2040, "bf16", 0, 256), (6200, 2048, 2040, "bf16", 1, 256), (3100, 2048, 2040, "f16", 0, 256),
             (2100, 2048, 2040, "f32", 0, 256), (8200, 2050, 2051, "bf16", 0, 256), (8200, 2050, 2051, "f16", 3, 256), (8200, 2050, 2051, "f32", 1, 256),
             (4096, 300, 333, "bf16", 0, 128), (4096, 300, 333, "f16", 0, 128), (4096, 300, 333, "f32", 0, 128), (4100, 304, 332, "bf16", 0, 128)]


@pytest.mark.parametrize("M, N, K, dtype, start, tile", GRADIENTS)
def test_weight_gradients(M, N, K, dtype, start, tile):
    plan = hip.lib().ifl_block8_wgrad_plan(M, N, K, TYPE[dtype])
    assert plan & 0xffff == tile and plan >> 16 > 1
    g = gen(M + N)
    # gradients that need all of their type's terms; a checkpoint sparse enough for sums of their magnitudes below 2^24
    most, share = {"bf16": (127, 1.0), "f16": (2047, 0.3), "f32": ((1 << 18) - 1, 0.004)}[dtype]
    store = torch.full((start + M * N + 8,), float("nan"), device="cuda", dtype=DT[dtype])
    dy = store[start:start + M * N].view(M, N)
    dy.copy_(ints(g, M, N, most))
    x = ints(g, M, K, 1) * (torch.rand(M, K, generator=g, device="cuda") < share) * torch.pow(2.0, torch.randint(0, 2, (M, 1), generator=g, device="cuda").float())
    assert float((dy.float().abs().t() @ x.abs()).max()) < 1 << 24
    q = block8.quantize(x, "e5m2" if K % 2 else "e4m3")
    assert torch.equal(R.of(q), x.double())
    ref, sums = dy.double().t() @ x.double(), dy.double().sum(0)
    for out in {torch.float32, DT[dtype]}:
        dw, _ = block8.weight_grad(dy, q, out)
        assert torch.equal(dw, ref.to(out))
    dw, db = block8.weight_grad(dy, q, torch.float32, torch.float32)
    assert torch.equal(dw, ref.float())
    assert bool(((db.double() - sums).abs() <= M * 2.0 ** -24 * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("dtype, exact", [("f32", True), ("bf16", True), ("bf16", False), ("f16", True)])
def test_layer(dtype, exact):
    """linear8 where both products and the weight gradient go to the large tiles."""
    M, N, K = 6200, 2048, 2040
    L = hip.lib()
    assert L.ifl_block8_matmul_plan(M, N, K) & 0xffff == 256 and L.ifl_block8_matmul_plan(M, K, N) & 0xffff == 256
    assert L.ifl_block8_wgrad_plan(M, N, K, TYPE[dtype]) & 0xffff == 256
    g = gen(5)
    x, w, gy, b = (t.to(DT[dtype]) for t in (ints(g, M, K, 3), ints(g, N, K, 3), ints(g, M, N, 3), ints(g, 1, N, 7)[0]))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = train_ops.linear8(*leaves, exact=exact)
    y.backward(gy)
    x, w, gy, b = (t.double() for t in (x, w, gy, b))
    for got, ref in ((y.detach(), x @ w.t() + b), (leaves[0].grad, gy @ w), (leaves[1].grad, gy.t() @ x), (leaves[2].grad, gy.sum(0))):
        assert float(ref.abs().max()) < 1 << 24
        assert torch.equal(got, ref.to(DT[dtype]))
