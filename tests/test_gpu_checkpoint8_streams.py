"""A checkpoint's channel factors, made at their first use, where another stream or a captured graph uses them first."""
import pytest
import torch

from interflow_amd import train_ops

pytestmark = pytest.mark.gpu


def checkpoint():
    g = torch.Generator().manual_seed(70)
    x = torch.nn.functional.pad(torch.randn(2, 6, 7, 64, generator=g), (0, 0, 1, 1, 1, 1)).cuda()
    bias, logs = torch.randn(64, generator=g).cuda(), 0.3 * torch.randn(64, generator=g).cuda()
    make = lambda: train_ops.an_relu8_ring(x, bias, logs)[1]      # noqa: E731
    want = make().restore()
    return make(), want


def test_first_use_on_a_stream_that_is_behind():
    ck, want = checkpoint()
    torch.cuda.synchronize()
    late, early = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(late):
        torch.cuda._sleep(100_000_000)                                      # (some 50 ms)
        first = ck.restore()
    with torch.cuda.stream(early):
        second = ck.restore()
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)


def test_first_use_in_a_captured_graph():
    ck, want = checkpoint()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.restore()
    assert torch.equal(ck.restore(), want)                                  # nothing was replayed yet
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del graph, out
    junk = torch.full((1 << 20,), float("nan"), device="cuda")
    assert torch.equal(ck.restore(), want) and junk.isnan().all()


def test_use_in_a_captured_graph_after_the_first():
    ck, want = checkpoint()
    ck.restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.restore()
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_logs_of_inference_mode():
    with torch.inference_mode():
        ck, want = checkpoint()
        assert torch.equal(ck.restore(), want)
