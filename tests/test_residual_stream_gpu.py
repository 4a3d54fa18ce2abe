"""The operators around the mixers as a model uses them: stream -> norm -> mixer -> stream ... -> norm -> head.  Each step is checked
against the formula in 64 bits of what the step before really gave; the bounds are those of the operators' own tests."""
import pytest
import torch

from quamba_amd import QRMSNorm, W4A8B16O16Linear, W8A8B16O16Linear, ops
from test_add_rmsnorm_gpu import check as check_norm
from test_add_rmsnorm_gpu import reference as norm_reference
from test_mixer_gpu import D_MODEL, _mixer
from test_token_logprobs_gpu import check as check_logprobs

pytestmark = pytest.mark.gpu
VOCAB = 1003


def _norm(dev, seed, output_scale, post=False, **more):
    g = torch.Generator().manual_seed(seed)
    n = QRMSNorm(D_MODEL, post_norm=post, device=dev, **more)
    n.weight = (1 + 0.2 * torch.randn(D_MODEL, generator=g)).half().to(dev)
    if post:
        n.post_weight = (1 + 0.2 * torch.randn(D_MODEL, generator=g)).half().to(dev)
    n.output_scale = output_scale
    return n


def _head(dev, seed=3):
    h = W8A8B16O16Linear(D_MODEL, VOCAB, device=dev)
    g = torch.Generator().manual_seed(seed)
    h._set_weight(torch.randint(-127, 128, (VOCAB, D_MODEL), generator=g).to(dev))
    h.a, h.b = torch.tensor([[0.03]], device=dev), torch.tensor([[0.002]], device=dev)
    h.alpha = 0.03 * 0.002
    return h


def _rows(t):
    return t.flatten(0, -2)


def _checked_norm(n, x, residual, got, **more):
    """got: what n gave with prenorm"""
    y, scales, stream = got if len(got) == 3 else (got[0], None, got[1])
    want = norm_reference(_rows(x), n.weight, n.eps, None if residual is None else _rows(residual), n.post_weight, **more)
    check_norm((_rows(y), _rows(stream), None if scales is None else scales.reshape(-1)), want, x, n.output_scale)


@pytest.mark.parametrize("batch,seqlen", [(2, 33), (1, 300)])
def test_two_blocks_and_a_head(dev, batch, seqlen):
    mixers = [_mixer(dev, seed=i)[0] for i in range(2)]
    norms = [_norm(dev, 0, 0.03), _norm(dev, 1, 0.025, post=True), _norm(dev, 2, None)]
    head = _head(dev)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(batch, seqlen, D_MODEL, generator=g).half().to(dev)
    tokens = torch.randint(-1, VOCAB, (batch, seqlen), generator=g).to(dev)

    got = norms[0](x, prenorm=True, residual_in_fp32=True)
    assert got[1].dtype == torch.float32
    _checked_norm(norms[0], x, None, got)
    stream = got[1]
    block = mixers[0](got[0])
    got = norms[1](block, stream, prenorm=True, residual_scale=0.5)
    _checked_norm(norms[1], block, stream, got, residual_scale=0.5)
    stream = got[1]
    block = mixers[1](got[0])
    last = norms[2](block, stream, prenorm=True)
    _checked_norm(norms[2], block, stream, last)
    hidden, scales, _ = last
    assert hidden.shape == x.shape and scales.shape == (batch, seqlen)
    # (without the stream the same codes)
    again = norms[2](block, stream)
    assert torch.equal(again[0], hidden) and torch.equal(again[1], scales)

    r = head.token_logprobs(hidden, tokens, top=1, x_scale=scales)
    assert r.logprobs.shape == (batch, seqlen) and r.top_tokens.shape == (batch, seqlen, 1)
    acc = (_rows(hidden).cpu().double() @ head.weight.cpu().double()[:, :VOCAB]).float()
    logits = scales.reshape(-1, 1).cpu() * (head.b.cpu() * acc)
    check_logprobs(ops.TokenLogprobs(r.logprobs.flatten(), r.entropy.flatten(), _rows(r.top_logprobs), _rows(r.top_tokens)), logits, tokens.flatten(), 1)
    # more alternatives: of the logits as forward rounds them
    many = head.token_logprobs(hidden, tokens, top=7, x_scale=scales)
    check_logprobs(ops.TokenLogprobs(many.logprobs.flatten(), many.entropy.flatten(), _rows(many.top_logprobs), _rows(many.top_tokens)), logits.half(),
                   tokens.flatten(), 7)
    # the layer's own scale: what forward's logits say, to their rounding
    plain, wide = head.token_logprobs(hidden, tokens), head(hidden).float()
    assert torch.allclose(plain.entropy, torch.distributions.Categorical(logits=wide).entropy(), rtol=2e-3, atol=2e-3)


def test_steps_captured_and_replayed(dev):
    """A decoding step of a block, its norms and the head as one graph: each replay against the eager step from the same states."""
    m = _mixer(dev, seed=4)[0]
    first, last, head, batch = _norm(dev, 0, 0.03), _norm(dev, 2, None), _head(dev), 3

    def step(x, tokens, states):
        h, stream = first(x, prenorm=True, residual_in_fp32=True)
        out, *_ = m.step(h, *states)
        h, s = last(out, stream)
        return head.token_logprobs(h, tokens, top=1, x_scale=s)

    x = torch.randn(batch, 1, D_MODEL, device=dev).half()
    tokens = torch.randint(0, VOCAB, (batch, 1), device=dev)
    held, eager = m.allocate_inference_cache(batch), m.allocate_inference_cache(batch)
    step(x, tokens, [s.clone() for s in held])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(x, tokens, held)
    for s in held:
        s.zero_()
    for i in range(4):
        x.copy_(torch.randn(batch, 1, D_MODEL, device=dev))
        tokens.random_(0, VOCAB)
        graph.replay()
        now = step(x, tokens, eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, now)), i
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), i


def test_head_of_4_bit_weights(dev):
    layer = torch.nn.Linear(256, 500, bias=False).half().to(dev)
    head = W4A8B16O16Linear.from_fp16(layer, torch.tensor(0.02))
    x = torch.randint(-127, 128, (2, 9, 256), dtype=torch.int8, device=dev)
    tokens = torch.randint(0, 500, (2, 9), device=dev)
    scales = torch.rand(2, 9, device=dev) * 0.05 + 0.01
    for top, x_scale in ((0, None), (3, scales)):
        r = head.token_logprobs(x, tokens, top, x_scale)
        s = x_scale.reshape(-1) if x_scale is not None else head.input_scale.reshape(1)
        logits = ops.w4a8o16_gemm(_rows(x), head.weight, s, head.s_channel, head.s_group, head.workspace, 18, head.size_n, head.size_k)[:, :500]
        check_logprobs(ops.TokenLogprobs(r.logprobs.flatten(), r.entropy.flatten(), _rows(r.top_logprobs), _rows(r.top_tokens)), logits, tokens.flatten(), top)
    assert torch.equal(head(x)[1, 3], ops.w4a8o16_gemm(_rows(x), head.weight, head.input_scale.reshape(1), head.s_channel, head.s_group, head.workspace, 18,
                                                       head.size_n, head.size_k)[12, :500])


def test_norm_module(dev):
    """Shapes, kinds of output and the state dict."""
    class Float(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.weight, self.eps = torch.nn.Parameter(1 + 0.1 * torch.randn(D_MODEL, device=dev)), 1e-6
    n = QRMSNorm.from_fp16(Float(), output_scale=0.04, post_layer=Float())
    x, r, gate = (torch.randn(2, 5, D_MODEL, device=dev).half() for _ in range(3))
    got = n(x, r, prenorm=True, gate=gate, gate_act="silu", residual_scale=0.3)
    assert got[0].dtype == torch.int8 and got[1].dtype == torch.float16
    _checked_norm(n, x, r, got, gate=_rows(gate), gate_act="silu", residual_scale=0.3)
    assert torch.equal(n(x, r, gate=gate, gate_act="silu", residual_scale=0.3), got[0])
    other = QRMSNorm(D_MODEL, eps=1e-6, post_norm=True, device=dev)
    other.load_state_dict(n.state_dict())
    assert other.output_scale == 0.04 and torch.equal(other(x, r), n(x, r))
    dynamic = QRMSNorm.from_fp16(Float())
    codes, scales = dynamic(x)
    assert codes.shape == x.shape and scales.shape == (2, 5)
    again = QRMSNorm(D_MODEL, device=dev)
    again.load_state_dict(dynamic.state_dict())
    assert again.output_scale is None
    wide = QRMSNorm.from_fp16(Float(), use_float_output=True)
    assert wide(x[0, 0]).shape == (D_MODEL,) and wide(x).dtype == torch.float16
    # a stream in one piece of memory that lies across the rows' order
    turned = torch.randn(5, 2, D_MODEL, device=dev).half().transpose(0, 1)
    assert torch.equal(wide(turned), wide(turned.contiguous()))
    for bad in (dict(residual=r[:1]), dict(gate=gate[:1]), dict(gate=gate[..., :8])):
        with pytest.raises(RuntimeError):
            n(x, **bad)
    head = _head(dev)
    codes = torch.zeros(2, 5, D_MODEL, dtype=torch.int8, device=dev)
    for bad in (dict(tokens=torch.zeros(10, dtype=torch.int64, device=dev)), dict(tokens=torch.zeros(2, 5, dtype=torch.int64, device=dev), x_scale=scales[:1])):
        with pytest.raises(RuntimeError):
            head.token_logprobs(codes, **bad)
