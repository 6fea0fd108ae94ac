"""8-bit blocks behind 2^31 elements, with values that make the far ones decide the result."""
import pytest
import torch

from interflow_amd import block8, train_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2])
def test_longest_rows(rows):
    """The most columns that are accepted: every value of e4m3's whole numbers up to 8 comes back."""
    cols = 0x7FFFFC00
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randint(-8, 9, (rows, cols), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    q = block8.quantize(x)
    assert torch.equal(block8.dequantize(q, torch.bfloat16), x)


# 2.3e9 values: rows from 65536 on lie behind 2^31 of them
ROWS, COLS, FAR = 70001, 32768, 65536
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def whole(seed, rows, cols, most, dtype):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda", dtype=torch.int8).to(dtype)


def test_every_row_of_a_large_matrix():
    """Quantized, restored and multiplied; whole numbers, so every sum is exact and every row counts by itself."""
    x = whole(1, ROWS, COLS, 2, torch.bfloat16)
    q = block8.quantize(x)
    assert torch.equal(block8.dequantize(q, torch.bfloat16), x)
    w = whole(2, 64, COLS, 2, torch.bfloat16)
    wq = block8.quantize(w)
    y, z = block8.matmul(q, wq, dtype=torch.float32), block8.linear(x, wq)
    t = block8.matmul(wq, q, dtype=torch.float32)                            # (it is the n side that is large)
    for at in range(0, ROWS, 8192):
        ref = x[at:at + 8192].float() @ w.float().t()
        assert torch.equal(y[at:at + 8192], ref) and torch.equal(t[:, at:at + 8192], ref.t()) and torch.equal(z[at:at + 8192], ref.bfloat16())


def test_every_row_of_a_large_result():
    a, b = whole(3, ROWS, 128, 3, torch.float32), whole(4, COLS, 128, 3, torch.float32)
    y = block8.matmul(block8.quantize(a), block8.quantize(b), dtype=torch.bfloat16)
    for at in range(0, ROWS, 8192):
        assert torch.equal(y[at:at + 8192], (a[at:at + 8192] @ b.t()).bfloat16())


def test_weight_gradient_of_far_codes():
    """Only rows behind 2^31 codes have gradients."""
    q = block8.quantize(whole(5, ROWS, COLS, 1, torch.bfloat16))
    dy = whole(6, ROWS, 8, 3, torch.bfloat16)
    dy[:FAR] = 0
    x = block8.dequantize(block8.Block8(q.codes[FAR:], q.scales[FAR:]))
    for dtype in DT.values():
        dw, db = block8.weight_grad(dy.to(dtype), q, bias_dtype=torch.float32)
        assert torch.equal(dw, dy[FAR:].float().t() @ x) and torch.equal(db, dy.float().sum(0)) and bool(dw.any())


@pytest.mark.parametrize("dtype", list(DT))
def test_weight_gradient_of_far_gradients(dtype):
    """Only what lies behind 2^31 gradients is not zero (bf16: read in place)."""
    dy = whole(7, ROWS, COLS, 3, DT[dtype])
    dy[:FAR] = 0
    x = whole(8, ROWS, 8, 3, torch.float32)
    dw, db = block8.weight_grad(dy, block8.quantize(x), bias_dtype=torch.float32)
    far = dy[FAR:].float()
    assert torch.equal(dw, far.t() @ x[FAR:]) and torch.equal(db, far.sum(0)) and bool(dw.any())


def test_every_pixel_of_a_large_activation():
    """ActNorm + ReLU: outputs and dx everywhere, sums over gradients of far pixels only."""
    H, C = 1500, 1024
    first = (1 << 31) // (H * C) + 1                                         # lines behind 2^31 elements
    g = torch.Generator("cuda").manual_seed(9)
    draw = lambda: torch.randint(-8, 9, (1, H, H, C), generator=g, device="cuda", dtype=torch.int8).float()      # noqa: E731
    x, gy = draw(), draw()
    gy[:, :first] = 0
    bias = torch.randint(-2, 3, (C,), generator=g, device="cuda").float().requires_grad_()
    logs = torch.zeros(C, device="cuda", requires_grad=True)
    leaf = x.detach().requires_grad_()
    y, ck = train_ops.an_relu8_ring(leaf, bias, logs)
    y.backward(gy)
    inner = torch.zeros(H, H, 1, device="cuda")
    inner[1:-1, 1:-1] = 1
    db, dl = torch.zeros(C, device="cuda", dtype=torch.float64), torch.zeros(C, device="cuda", dtype=torch.float64)
    back = ck.restore()
    for at in range(0, H, 100):
        part = slice(at, at + 100)
        v = (x[0, part] + bias.detach()).relu() * inner[part]
        d = torch.where(v > 0, gy[0, part], 0.0)
        assert torch.equal(y[0, part], v) and torch.equal(back[0, part], v) and torch.equal(leaf.grad[0, part], d), at
        db += d.double().sum((0, 1))
        dl += (d * v).double().sum((0, 1))
    # (sums of whole numbers below 2^24: exact)
    assert torch.equal(bias.grad.double(), db) and torch.equal(logs.grad.double(), dl) and bool(db.any())
