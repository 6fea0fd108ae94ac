"""8-bit operators on tensors as programs have them: transposed, sliced, strided, odd starts, rows of none; whole numbers, so results are exact."""
import random

import pytest
import torch

from interflow_amd import block8, train_ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [0, 1, 2, 7, 8, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 511, 640]


def lay(rng, t):
    """The values of t [rows, cols] in memory of some other order, NaN around them."""
    r, c = t.shape
    kind = rng.choice(["plain", "transposed", "slice", "odd start", "every second row", "every second column"])
    if kind == "plain":
        return t
    if kind == "transposed":
        return t.t().contiguous().t()
    if kind == "slice":
        big = torch.full((r + 3, c + 11), float("nan"), device="cuda", dtype=t.dtype)
        v = big[2:2 + r, 5:5 + c]
    elif kind == "odd start":
        v = torch.full((r * c + 9,), float("nan"), device="cuda", dtype=t.dtype)[1:1 + r * c].view(r, c)
    elif kind == "every second row":
        v = torch.full((2 * r, c), float("nan"), device="cuda", dtype=t.dtype)[::2]
    else:
        v = torch.full((r, 2 * c), float("nan"), device="cuda", dtype=t.dtype)[:, ::2]
    v.copy_(t)
    return v


@pytest.mark.parametrize("seed", range(60))
def test_layouts(seed):
    rng, g = random.Random(seed), torch.Generator("cuda").manual_seed(seed)
    M, N, K = rng.choice(SIZES), rng.choice(SIZES[1:]), rng.choice(SIZES[1:])
    dt, wt, bt = (rng.choice(TYPES) for _ in range(3))
    exact = rng.random() < 0.6

    def ints(rows, cols, dtype, most=3):
        return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda").to(dtype)
    x, w, gy, bias = lay(rng, ints(M, K, dt)), lay(rng, ints(N, K, wt)), lay(rng, ints(M, N, dt)), ints(1, N, bt, 7)[0]
    X, W, G = x.double(), w.double(), gy.double()
    leaves = [t.detach().requires_grad_() for t in (x, w, bias)]
    y = train_ops.linear8(*leaves, rng.choice(["e4m3", "e5m2"]), exact)
    y.backward(gy)
    ref = X @ W.t() + bias.double()
    assert torch.equal(y.detach(), ref.to(dt))
    assert torch.equal(leaves[0].grad, (G @ W).to(dt))
    assert torch.equal(leaves[1].grad, (G.t() @ X).to(wt))
    assert torch.equal(leaves[2].grad, G.sum(0).to(bt))
    a, b = block8.quantize(x, rng.choice(["e4m3", "e5m2"])), block8.quantize(w, rng.choice(["e4m3", "e5m2"]))
    if rng.random() < 0.5:
        a = block8.Block8(a.codes.contiguous(), a.scales.contiguous())
    assert torch.equal(block8.dequantize(a).double(), X)
    assert torch.equal(block8.matmul(a, b, bias, dt, exact), ref.to(dt))
    assert torch.equal(block8.linear(x, b, bias, exact), ref.to(dt))
    dw, db = block8.weight_grad(gy, a, wt, bt)
    assert torch.equal(dw, (G.t() @ X).to(wt)) and torch.equal(db, G.sum(0).to(bt))
