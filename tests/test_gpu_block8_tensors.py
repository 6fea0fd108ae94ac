"""Block8 of a caller's tensors: what the caller does to them afterwards counts."""
import pytest
import torch

from interflow_amd import block8

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def results(q, w, dy):
    return [block8.dequantize(q), block8.matmul(q, w), block8.matmul(w, q), block8.linear(block8.dequantize(w), q), block8.weight_grad(dy, q)[0]]


@pytest.mark.parametrize("rows", [1, 30])
def test_tensors_with_other_memory(rows):
    """Given other memory, as a module that moves its parameters does it; then rows another distance apart."""
    old, new, w, dy = block8.quantize(rand(1, rows, 300)), block8.quantize(rand(2, rows, 300)), block8.quantize(rand(3, 40, 300)), rand(4, rows, 20)
    codes, scales = old.codes.clone(), old.scales.clone()
    q = block8.Block8(codes, scales)
    want = results(old, w, dy)
    assert all(torch.equal(a, b) for a, b in zip(results(q, w, dy), want))
    kept = codes.data, scales.data                                           # (the first memory stays as it was)
    codes.data, scales.data = new.codes.clone(), new.scales.clone()
    want = results(new, w, dy)
    assert all(torch.equal(a, b) for a, b in zip(results(q, w, dy), want))
    wide = torch.zeros(rows, 320, dtype=torch.uint8, device="cuda")
    wide[:, :300] = old.codes.view(torch.uint8)
    codes.data, scales.data = wide.view(old.codes.dtype)[:, :300], kept[1]
    want = results(old, w, dy)
    assert all(torch.equal(a, b) for a, b in zip(results(q, w, dy), want))


def test_columns_that_are_not_contiguous():
    """They are copied in each call, not once: a change in place is seen."""
    q, w, dy = block8.quantize(rand(5, 30, 300)), block8.quantize(rand(6, 40, 300)), rand(7, 30, 20)
    codes, scales = q.codes.view(torch.uint8).t().contiguous().t().view(q.codes.dtype), q.scales.view(torch.uint8).t().contiguous().t().view(q.scales.dtype)
    p = block8.Block8(codes, scales)
    assert all(torch.equal(a, b) for a, b in zip(results(p, w, dy), results(q, w, dy)))
    other = block8.quantize(rand(8, 30, 300))
    codes.view(torch.uint8).copy_(other.codes.view(torch.uint8))
    scales.view(torch.uint8).copy_(other.scales.view(torch.uint8))
    assert all(torch.equal(a, b) for a, b in zip(results(p, w, dy), results(other, w, dy)))


def test_tensors_of_another_shape_are_refused():
    q, w, dy = block8.quantize(rand(9, 30, 300)), block8.quantize(rand(10, 40, 300)), rand(11, 30, 20)
    codes, scales = q.codes.clone(), q.scales.clone()
    p = block8.Block8(codes, scales)
    codes.data = codes.data[:20]
    for call in (lambda: block8.dequantize(p), lambda: block8.matmul(p, w), lambda: block8.matmul(w, p), lambda: block8.linear(rand(12, 5, 300), p), lambda: block8.weight_grad(dy, p)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("cols", [640, 150])
def test_aligned_once(cols):
    """Weights whose rows are not whole 16 and 4 bytes: their aligned form gives the same results and is not copied again."""
    w, x = block8.quantize(rand(13, 40, cols)), rand(14, 20, cols)
    p = block8.Block8(w.codes.contiguous(), w.scales.contiguous())
    a = p.aligned()
    assert a is not p and a.aligned() is a and w.aligned() is w
    assert torch.equal(a.codes.view(torch.uint8), p.codes.view(torch.uint8)) and torch.equal(a.scales.view(torch.uint8), p.scales.view(torch.uint8))
    assert torch.equal(block8.linear(x, a), block8.linear(x, p)) and torch.equal(block8.linear(x, a), block8.linear(x, w))
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    block8.linear(x[:1], a)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before + 1          # (its result; the launch quantizes the row itself)


def test_tensors_of_another_type_are_refused():
    q = block8.quantize(rand(15, 30, 300))
    codes, scales = q.codes.clone(), q.scales.clone()
    p = block8.Block8(codes, scales)
    codes.data = codes.view(torch.uint8).view(torch.float8_e5m2)
    with pytest.raises(RuntimeError):
        block8.dequantize(p)
