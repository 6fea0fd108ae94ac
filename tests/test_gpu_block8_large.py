"""8-bit blocks behind 2^31 elements, with values that make the far ones decide the result."""
import pytest
import torch

from interflow_amd import block8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2])
def test_longest_rows(rows):
    """The most columns that are accepted: every value of e4m3's whole numbers up to 8 comes back."""
    cols = 0x7FFFFC00
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randint(-8, 9, (rows, cols), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    q = block8.quantize(x)
    assert torch.equal(block8.dequantize(q, torch.bfloat16), x)
