"""Sums of the 8-bit ActNorm + ReLU's backward pass over many pixels."""
import pytest
import torch

from interflow_amd import train_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("c", [1 + 0.49 * 2.0 ** -16, 1 + 0.3 * 2.0 ** -17, 1.1])
def test_sums_of_equal_gradients(c):
    """Every addition of a long row rounds the same way.  Here 241 pixels to a thread in rows of 16 (16 additions, then 16), two threads to
    a workgroup in LDS (3), 1023 workgroups in 64 rows of four (4 and 2), joined in pairs (6): 47 additions at most on a value's way,
    each off by at most 2^-24 of what is there."""
    H, C = 700, 1024
    x = torch.zeros(1, H + 2, H + 2, C, device="cuda")
    x[:, 1:-1, 1:-1] = 1.0
    bias, logs = torch.zeros(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    g = torch.zeros_like(x)
    g[:, 1:-1, 1:-1] = c
    y, _ = train_ops.an_relu8_ring(x, bias, logs)
    y.backward(g)
    want = H * H * float(torch.tensor(c))
    for got in (bias.grad, logs.grad):
        assert float((got.double() - want).abs().max()) <= 47 * 2.0 ** -24 * want
