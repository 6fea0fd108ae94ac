"""The weight gradient of a convolution whose input is kept as an 8-bit checkpoint, against its formula in float64."""
import pytest
import torch
import torch.nn.functional as F

from interflow_amd import train_ops

pytestmark = pytest.mark.gpu


def ring(x):
    return F.pad(x, (0, 0, 1, 1, 1, 1))


@pytest.mark.parametrize("k, cin, cout, B, H, W", [(1, 64, 64, 2, 9, 8), (1, 128, 96, 1, 13, 7), (1, 32, 20, 3, 4, 40), (3, 64, 24, 2, 9, 8), (3, 96, 64, 1, 20, 12)])
def test_weight_gradient(k, cin, cout, B, H, W):
    g = torch.Generator().manual_seed(k + cin)
    rand = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    x, bias, logs = ring(rand(B, H, W, cin)).cuda(), rand(cin).cuda(), 0.3 * rand(cin).cuda()
    w, b = rand(cout, cin, k, k).cuda().requires_grad_(), rand(cout).cuda().requires_grad_()
    a, ck = train_ops.an_relu8_ring(x, bias, logs)
    y = train_ops.conv2d_ring([a], [cin], w, b, [ck])
    gy = F.pad(rand(B, H, W, cout), (0, train_ops.pad32(cout) - cout, 1, 1, 1, 1)).cuda()
    y.backward(gy)
    # the activation that the checkpoint stands for: its values, exact, times exp(logs)
    v = ck.codes.float().double() * torch.pow(2.0, ck.scales.view(torch.uint8).double() - 127).repeat_interleave(128, 3)[..., :cin]
    act = (v * logs.double().exp())[:, 1:-1, 1:-1].permute(0, 3, 1, 2).cpu()
    d = gy[:, 1:-1, 1:-1, :cout].double().permute(0, 3, 1, 2).cpu()

    def formula(act, d):
        weight = torch.zeros(cout, cin, k, k, dtype=torch.float64, requires_grad=True)
        return torch.autograd.grad(F.conv2d(act, weight, padding=k // 2), weight, d)[0]
    # n products, each sum within n 2^-23 of their magnitudes; a factor exp(logs) within a few units of its last place
    err = (B * H * W * 2.0 ** -23 + 2.0 ** -20) * formula(act.abs(), d.abs())
    assert bool(((w.grad.double().cpu() - formula(act, d)).abs() <= err).all())
    assert bool(((b.grad.double().cpu() - d.sum((0, 2, 3))).abs() <= B * H * W * 2.0 ** -23 * d.abs().sum((0, 2, 3))).all())
