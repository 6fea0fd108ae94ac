"""The 8-bit block format's reference against torch's conversions, and the operators' refusals: no GPU needed."""
import math

import pytest
import torch

from interflow_amd import block8, hip, train_flow, train_ops
from tests import _block8_ref as R


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_reference_rounds_as_torchs_conversion(fmt):
    """Every value a block can hold after scaling: the reference's rounding against torch's float8 conversion."""
    dt, _, _, top = R.FORMATS[fmt]
    g = torch.Generator().manual_seed(1)
    big = 1.75 * 2.0 ** top
    x = torch.cat([torch.randn(64, 128, generator=g), torch.randn(64, 128, generator=g) * torch.exp(8 * torch.randn(64, 128, generator=g))])
    every = torch.arange(0, 256, dtype=torch.uint8).view(dt).float()                       # all codes, and the ties between neighbours
    every = every[every.isfinite() & (every.abs() <= big)].unique()
    ties = (every[1:] + every[:-1]) / 2
    pool = torch.cat([every, ties])
    pool = torch.nn.functional.pad(pool, (0, -pool.numel() % 127)).view(-1, 127)
    x = torch.cat([x, torch.cat([torch.full((pool.shape[0], 1), big), pool], 1)])
    codes, e = R.split(x, fmt)
    scaled = (x.double() * R.two_to(-e)).float()
    assert torch.equal(codes.float(), scaled.to(dt).float())
    assert bool((scaled.abs() <= big).all())
    m = x.abs().amax(1).double()
    assert bool((m <= big * R.two_to(e[:, 0])).all()) and bool(((m > big * R.two_to(e[:, 0] - 1)) | (e[:, 0] == -126)).all())


def test_reference_special_values():
    x = torch.tensor([[0.0, -0.0, math.nan, math.inf, -math.inf, 448.0, 1.0]])
    v = R.values(x, "e4m3")
    assert v[0, 5] == 448 and v[0, 6] == 1 and bool(v[0, 2:5].isnan().all())
    v = R.values(x, "e5m2")
    assert v[0, 3] == math.inf and v[0, 4] == -math.inf and v[0, 2].isnan() and v[0, 5] == 448
    assert R.split(torch.zeros(1, 5), "e4m3")[1].item() == -126
    assert R.values(torch.tensor([[1.0, 1e-9]]), "e4m3")[0, 1] == 0
    assert R.values(torch.tensor([[1.0, 1e-9]]), "e4m3", keep_positive=True)[0, 1] > 0


def test_operators_refuse_host_tensors():
    x = torch.zeros(4, 64)
    with pytest.raises(hip.InterflowHipError):
        block8.quantize(x)
    with pytest.raises(hip.InterflowHipError):
        block8.Block8(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    with pytest.raises(hip.InterflowHipError):
        train_ops.linear8(x, torch.zeros(8, 64))
    with pytest.raises(hip.InterflowHipError):
        train_ops.an_relu8_ring(torch.zeros(1, 4, 4, 32), torch.zeros(32), torch.zeros(32))
    with pytest.raises(TypeError):
        block8.quantize([1.0])
    with pytest.raises(TypeError):
        block8.dequantize(x)
    with pytest.raises(TypeError):
        block8.matmul(x, x)


def test_checkpoint_switch():
    prev = train_flow.set_activation_checkpoints()
    try:
        assert train_flow.set_activation_checkpoints(8) == prev
        assert train_flow.set_activation_checkpoints() == 8
        with pytest.raises(ValueError):
            train_flow.set_activation_checkpoints(16)
        assert train_flow.set_activation_checkpoints(32) == 8
    finally:
        train_flow.set_activation_checkpoints(prev)


@pytest.mark.parametrize("call, args", [
    # (types and formats outside the lists, shapes below one, rows closer than they are long, null pointers: all before any launch)
    ("ifl_block8_quantize", (16, 3, 64, 1, 16, 64, 16, 1, 1, 64, 0, None)),
    ("ifl_block8_quantize", (16, 0, 64, 1, 16, 64, 16, 1, 1, 64, 2, None)),
    ("ifl_block8_quantize", (16, 0, 64, 1, 16, 64, 16, 1, 1, 0, 0, None)),
    ("ifl_block8_quantize", (16, 0, 64, 1, 16, 64, 16, 1, -1, 64, 0, None)),
    ("ifl_block8_quantize", (16, 0, 64, 1, 16, 63, 16, 1, 1, 64, 0, None)),
    ("ifl_block8_quantize", (16, 0, 64, 1, 16, 129, 16, 1, 1, 129, 0, None)),
    ("ifl_block8_quantize", (16, 0, 64, 2, 16, 64, 16, 1, 2, 64, 0, None)),
    ("ifl_block8_quantize", (None, 0, 64, 1, 16, 64, 16, 1, 1, 64, 0, None)),
    ("ifl_block8_dequantize", (16, 63, 16, 1, 0, None, 16, 0, 64, 1, 64, None)),
    ("ifl_block8_dequantize", (16, 64, 16, 1, 0, None, 16, 3, 64, 1, 64, None)),
    ("ifl_block8_dequantize", (16, 64, 16, 1, 0, None, None, 0, 64, 1, 64, None)),
    ("ifl_block8_matmul", (16, 64, 16, 4, 0, 16, 64, 16, 4, 2, None, 0, 16, 0, 8, None, 1, 8, 64, None)),
    ("ifl_block8_matmul", (16, 72, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 8, None, 1, 8, 64, None)),
    ("ifl_block8_matmul", (8, 64, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 8, None, 1, 8, 64, None)),
    ("ifl_block8_matmul", (16, 64, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 7, None, 1, 8, 64, None)),
    ("ifl_block8_matmul", (16, 64, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 8, None, 1, 0, 64, None)),
    ("ifl_block8_wgrad", (16, 0, 8, 16, 64, 16, 1, 0, None, None, 0, 64, None, 0, None, 4, 8, 64, None)),
    ("ifl_block8_wgrad", (16, 0, 7, 16, 64, 16, 1, 0, None, 16, 0, 64, None, 0, 16, 4, 8, 64, None)),
    ("ifl_block8_wgrad", (16, 5, 8, 16, 64, 16, 1, 0, None, 16, 0, 64, None, 0, None, 4, 8, 64, None)),
    ("ifl_block8_wgrad", (16, 0, 8, 16, 64, 16, 1, 0, None, 16, 0, 64, None, 0, None, 4, 8, 64, None)),
    ("ifl_block8_wgrad", (16, 0, 8, 8, 64, 16, 1, 0, None, 16, 0, 64, None, 0, 16, 4, 8, 64, None)),
    ("ifl_block8_wgrad", (16, 0, 8, 16, 72, 16, 1, 0, None, 16, 0, 64, None, 0, 16, 4, 8, 64, None)),
    ("ifl_block8_linear", (16, 3, 64, 16, 64, 16, 4, 0, None, 0, 16, 8, 16, 1, 8, 64, None)),
    ("ifl_block8_linear", (16, 0, 64, 16, 64, 16, 4, 2, None, 0, 16, 8, 16, 1, 8, 64, None)),
    ("ifl_block8_linear", (None, 0, 64, 16, 64, 16, 4, 0, None, 0, 16, 8, 16, 1, 8, 64, None)),
    ("ifl_block8_linear", (16, 0, 63, 16, 64, 16, 4, 0, None, 0, 16, 8, 16, 2, 8, 64, None)),
    ("ifl_block8_linear", (16, 0, 64, 16, 64, 16, 4, 0, None, 0, 16, 7, 16, 1, 8, 64, None)),
    ("ifl_block8_linear", (16, 0, 64, 16, 64, 16, 4, 0, None, 0, 16, 8, None, 17, 8, 64, None)),
    ("ifl_block8_linear", (16, 0, 64, 8, 64, 16, 4, 0, None, 0, 16, 8, 16, 1, 8, 64, None)),
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, None, 4, 8, 64, None)),
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 8, 4, 8, 64, None)),
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, 4, 0, 64, None)),
    ("ifl_linear8_fwd", (16, 3, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, 4, 8, 64, None)),
    ("ifl_linear8_fwd", (None, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, 4, 8, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 8, 16, 16, 16, 0, 64, 1, 0, None, 16, None, 0, None, 4, 8, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 8, 16, 16, 16, 0, 64, 1, 0, None, 16, None, 0, 16, 4, 8, 0, None)),
    ("ifl_linear8_bwd", (16, 3, 8, 16, 16, 16, 0, 64, 1, 0, None, 16, None, 0, 16, 4, 8, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 7, 16, 16, 16, 0, 64, 1, 0, None, 16, None, 0, 16, 4, 8, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 8, 16, 16, 16, 0, 64, 1, 2, 16, None, None, 0, 16, 4, 8, 64, None)),
    ("ifl_linear8_bwd", (None, 0, 8, 16, 16, 16, 0, 64, 1, 0, None, 16, None, 0, 16, 4, 8, 64, None)),
    ("ifl_an_relu8_fwd", (16, 16, 16, 16, 16, 16, 0, 4, 4, 64, None)),
    ("ifl_an_relu8_fwd", (4, 16, 16, 16, 16, 16, 1, 4, 4, 64, None)),
    ("ifl_an_relu8_bwd", (16, 16, 16, 16, 16, None, 16, 16, 1, 4, 4, 64, None)),
])
def test_library_refuses(call, args):
    with pytest.raises(AssertionError):
        hip.check(getattr(hip.lib(), call)(*args), call)


@pytest.mark.parametrize("C", [0, 31, 48, 1056])
def test_library_refuses_channel_counts(C):
    with pytest.raises(NotImplementedError):
        hip.check(hip.lib().ifl_an_relu8_fwd(16, 16, 16, 16, 16, 16, 1, 4, 4, C, None), "ifl_an_relu8_fwd")


BIG = 1 << 30


@pytest.mark.parametrize("call, args", [
    # (sizes that a later step would refuse, after the first had run)
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, BIG, 8, 64, None)),
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, 4, 8, 1 << 23, None)),
    ("ifl_linear8_bwd", (16, 0, 8, 16, 16, 16, 0, 64, 1, 0, 16, None, None, 0, 16, BIG, 8, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 1 << 23, 16, 16, 16, 0, 64, 1, 0, 16, None, None, 0, 16, 4, 1 << 23, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 1 << 22, 16, 16, 16, 0, 64, 1, 0, 16, 16, None, 0, 16, 4, 1 << 22, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 8, 16, 16, 16, 0, 64, 1, 0, 16, 16, None, 0, 16, 4, 8, 1 << 22, None)),
    ("ifl_linear8_bwd", (16, 0, 1 << 23, 16, 16, 16, 0, 64, 1, 0, 16, None, 16, 0, 16, 4, 8, 64, None)),
])
def test_layer_refuses_before_any_launch(call, args):
    with pytest.raises(NotImplementedError):
        hip.check(getattr(hip.lib(), call)(*args), call)


def test_layer_refuses_what_its_backward_pass_would():
    for sizes, need in (((1 << 23, 8), (1, 0, 0)), ((1 << 22, 8), (0, 1, 0)), ((1 << 22, 8), (0, 0, 1)), ((8, 1 << 22), (0, 1, 0))):
        with pytest.raises(NotImplementedError):
            block8._backward_reaches(*sizes, *need)
    block8._backward_reaches((1 << 22) - 1, (1 << 22) - 1, 1, 1, 1)
    block8._backward_reaches(8, 1 << 22, 1, 0, 1)
    block8._backward_reaches((1 << 23) - 16, 1 << 22, 1, 0, 0)


@pytest.mark.parametrize("call, args", [
    # (more than 2^32 threads)
    ("ifl_block8_matmul", (16, 64, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 1 << 26, None, 1, 1 << 26, 64, None)),
    ("ifl_block8_matmul", (16, 64, 16, 4, 0, 16, 64, 16, 4, 0, None, 0, 16, 0, 1 << 17, None, 1 << 23, 1 << 17, 64, None)),
    ("ifl_block8_linear", (16, 0, 64, 16, 64, 16, 4, 0, None, 0, 16, 1 << 26, 16, 1, 1 << 26, 64, None)),
    ("ifl_linear8_fwd", (16, 0, 64, 1, 16, 0, 64, 1, None, 0, 16, 16, 16, 16, 4, 1 << 26, 64, None)),
    ("ifl_linear8_bwd", (16, 0, 64, 16, 16, 16, 0, 64, 1, 0, 16, None, None, 0, 16, 4, 64, 1 << 26, None)),
    ("ifl_block8_quantize", (16, 0, 1, 1 << 30, 16, 16, 16, 4, 1 << 30, 2, 0, None)),
])
def test_library_refuses_what_no_launch_holds(call, args):
    with pytest.raises(NotImplementedError):
        hip.check(getattr(hip.lib(), call)(*args), call)


def test_convolution_refuses_what_is_no_checkpoint_of_its_source():
    x, w = torch.zeros(1, 6, 6, 32), torch.zeros(8, 32, 1, 1)
    ck = train_ops.Checkpoint8(train_ops.Checkpoint8.room(x.shape, x), x.shape, torch.ones(32))
    for bad in (x, 8, "e4m3"):
        with pytest.raises(TypeError):
            train_ops.conv2d_ring([x], [32], w, checkpoints=[bad])
    for bad in ([], [ck, ck], [train_ops.Checkpoint8(ck.raw, torch.Size((1, 6, 5, 32)), torch.ones(32))], [train_ops.Checkpoint8(ck.raw.to("meta"), x.shape, torch.ones(32))]):
        with pytest.raises(AssertionError):
            train_ops.conv2d_ring([x], [32], w, checkpoints=bad)
