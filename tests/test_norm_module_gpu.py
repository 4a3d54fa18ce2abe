"""QRMSNorm with a stream that the caller holds, and its weights' types."""
import pytest
import torch

from quamba_amd import QRMSNorm

pytestmark = pytest.mark.gpu
DIM = 768


class Float(torch.nn.Module):
    def __init__(self, dev):
        super().__init__()
        self.weight, self.eps = torch.nn.Parameter(1 + 0.1 * torch.randn(DIM, device=dev)), 1e-5


@pytest.mark.parametrize("shape", [(DIM,), (5, DIM), (2, 7, DIM), (0, DIM)])
@pytest.mark.parametrize("output_scale", [None, 0.04])
def test_the_stream_in_place(dev, shape, output_scale):
    norm = QRMSNorm.from_fp16(Float(dev), output_scale)
    x, stream = torch.randn(shape, device=dev).half(), torch.randn(shape, device=dev)
    want = norm(x, stream, prenorm=True)
    place = torch.empty_like(stream)
    got = norm(x, stream, prenorm=True, residual_out=place)
    assert got[-1] is place and all(torch.equal(a, b) for a, b in zip(got, want))
    got = norm(x, stream, prenorm=True, residual_out=stream)
    assert got[-1] is stream and all(torch.equal(a, b) for a, b in zip(got, want))
    first = torch.empty_like(stream)
    got = norm(x, prenorm=True, residual_in_fp32=True, residual_out=first)
    assert torch.equal(first, x.float()) and got[-1] is first


def test_streams_that_do_not_fit(dev):
    norm = QRMSNorm.from_fp16(Float(dev))
    x, stream = torch.randn(2, 7, DIM, device=dev).half(), torch.randn(2, 7, DIM, device=dev)
    turned = torch.randn(7, 2, DIM, device=dev).transpose(0, 1)
    for bad in (dict(residual_out=stream[:1]), dict(residual_out=stream.half()), dict(residual_out=turned), dict(residual_out=stream.view(14, DIM)),
                dict(residual_out=x), dict(residual_out=stream, prenorm=False)):
        with pytest.raises(RuntimeError):
            norm(x, stream, **{"prenorm": True, **bad})
    # (what is read may lie in any order)
    want = norm(x, turned.contiguous(), prenorm=True)
    assert all(torch.equal(a, b) for a, b in zip(norm(x, turned, prenorm=True, residual_out=stream), want))


def test_captured_with_the_stream_in_place(dev):
    norm = QRMSNorm.from_fp16(Float(dev), 0.03)
    x, stream = torch.randn(3, 1, DIM, device=dev).half(), torch.zeros(3, 1, DIM, device=dev)
    norm(x, stream.clone(), prenorm=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, _ = norm(x, stream, prenorm=True, residual_out=stream)
    eager = stream.clone()
    for i in range(4):
        x.copy_(torch.randn(3, 1, DIM, device=dev))
        graph.replay()
        now, _ = norm(x, eager, prenorm=True, residual_out=eager)
        torch.cuda.synchronize()
        assert torch.equal(codes, now) and torch.equal(stream, eager), i


@pytest.mark.parametrize("rows,weights", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float32), (torch.float32, torch.float32)])
def test_weights_of_each_type(dev, rows, weights):
    layer, post = Float(dev), Float(dev)
    norm = QRMSNorm.from_fp16(layer, 0.04, post_layer=post, dtype=weights)
    x = torch.randn(4, DIM, device=dev).to(rows)
    by_hand = QRMSNorm(DIM, layer.eps, post_norm=True, device=dev, dtype=weights)
    by_hand.load_state_dict(norm.state_dict())
    assert norm.weight.dtype == weights and torch.equal(norm.weight, layer.weight.detach().to(weights))
    assert norm.post_weight.dtype == weights and torch.equal(norm.post_weight, post.weight.detach().to(weights))
    assert torch.equal(norm(x), by_hand(x)) and norm(x).dtype == torch.int8
    assert QRMSNorm.from_fp16(layer).weight.dtype == torch.float16
