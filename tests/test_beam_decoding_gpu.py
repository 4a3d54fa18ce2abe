"""A recurrent model decoded with beams: head in 4 bits, selection, states in their new order, a step of the mixer - as they are used together, and captured."""
import types

import pytest
import torch

from quamba_amd import MXFP4Linear, QRMSNorm, W4A8B16O16Linear, W8A8B16O16Linear, ops, reorder_cache
from test_mixer2_gpu import _mixer as mamba2
from test_mixer_gpu import _mixer as mamba1

pytestmark = pytest.mark.gpu
BATCH, BEAMS, STEPS, VOCAB = 3, 4, 6, 500


class Model:
    """Two mixers of random weights with norms between them"""

    def __init__(self, dev, kind):
        torch.manual_seed(3)
        self.mixers = [mamba1(dev, seed=s)[0] for s in range(2)] if kind == 1 else [mamba2(dev, seed=s)[0] for s in range(2)]
        d = self.mixers[0].d_model
        for i, m in enumerate(self.mixers):
            m.layer_idx = i
        self.embedding = torch.randn(VOCAB, d, device=dev).half()
        layers = [types.SimpleNamespace(weight=1 + 0.1 * torch.randn(d, device=dev), eps=1e-5) for _ in range(3)]
        self.norms = [QRMSNorm.from_fp16(n, output_scale=0.03) for n in layers[:2]] + [QRMSNorm.from_fp16(layers[2], use_float_output=True)]
        head = torch.nn.Linear(d, VOCAB, bias=False).half().to(dev)
        head.weight.data *= 4
        self.head = MXFP4Linear.from_fp16(head)

    def cache(self):
        return types.SimpleNamespace(key_value_memory_dict={i: m.allocate_inference_cache(BATCH * BEAMS) for i, m in enumerate(self.mixers)})

    def step(self, tokens, cache):
        """tokens (batch x beams,) -> (batch, beams, d)"""
        x, stream = self.embedding[tokens.clamp(min=0)].unsqueeze(1), None
        for i, m in enumerate(self.mixers):
            codes, stream = self.norms[i](x, stream, prenorm=True)
            x = m.step(codes, *cache.key_value_memory_dict[i])[0].view(BATCH * BEAMS, 1, -1)
        return self.norms[2](x, stream).view(BATCH, BEAMS, -1)


def plain_selection(logits, scores, count, done):
    """in torch's 64 bits, of equal ones the first"""
    offers = torch.log_softmax(logits.double(), -1) + scores.double()[..., None]
    offers.masked_fill_(done[..., None], float("-inf"))
    offers[..., 0] = torch.where(done, scores.double(), offers[..., 0])
    best, at = torch.sort(offers.flatten(1), dim=-1, descending=True, stable=True)
    best, at = best[:, :count], at[:, :count]
    parents, tokens = at // VOCAB, at % VOCAB
    return best.float(), torch.where(done.gather(1, parents), -1, tokens), parents


@pytest.mark.parametrize("kind", [1, 2])
def test_decoding_with_beams(dev, kind):
    """beams that end at token 7 stay as they are; against selection in torch and copies of the states"""
    model = Model(dev, kind)
    mine, theirs = model.cache(), model.cache()
    tokens = torch.randint(0, VOCAB, (BATCH,), device=dev)[:, None].expand(BATCH, BEAMS).reshape(-1)
    scores = torch.full((BATCH, BEAMS), float("-inf"), device=dev)
    scores[:, 0] = 0
    done = torch.zeros(BATCH, BEAMS, dtype=torch.bool, device=dev)
    changed = 0
    for _ in range(STEPS):
        hidden, again = model.step(tokens, mine), model.step(tokens, theirs)
        assert torch.equal(hidden, again)
        got = model.head.beam_search_step(hidden, scores, BEAMS, done)
        want = plain_selection(model.head(hidden), scores, BEAMS, done)
        assert torch.equal(got.tokens, want[1]) and torch.equal(got.parents, want[2])
        assert torch.allclose(got.scores, want[0], rtol=2.0 ** -23, atol=1e-6)
        reorder_cache(mine, got.parents)
        rows = (want[2] + BEAMS * torch.arange(BATCH, device=dev)[:, None]).reshape(-1)
        for i, states in theirs.key_value_memory_dict.items():
            for s, m in zip(states, mine.key_value_memory_dict[i]):
                s.copy_(s[rows])
                assert torch.equal(s, m)
        changed += int((got.parents != torch.arange(BEAMS, device=dev)).sum())
        scores, tokens = got.scores, got.tokens.view(-1)
        done = done.gather(1, got.parents) | (got.tokens == 7)
    assert changed > STEPS


def test_a_captured_step(dev):
    """selection, states and the mixers' step in one graph, replayed against the eager step"""
    model = Model(dev, 1)
    mine, theirs = model.cache(), model.cache()
    tokens, scores = torch.arange(BATCH * BEAMS, device=dev), torch.zeros(BATCH, BEAMS, device=dev)
    their_tokens, their_scores = tokens.clone(), scores.clone()

    def step(tokens, scores, cache):
        got = model.head.beam_search_step(model.step(tokens, cache), scores, BEAMS)
        reorder_cache(cache, got.parents)
        tokens.copy_(got.tokens.view(-1))
        scores.copy_(got.scores)
    for _ in range(2):
        step(tokens, scores, mine)
        step(their_tokens, their_scores, theirs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(tokens, scores, mine)
    for n in range(5):
        graph.replay()
        step(their_tokens, their_scores, theirs)
        torch.cuda.synchronize()
        assert torch.equal(tokens, their_tokens) and torch.equal(scores, their_scores), n
        for i, states in theirs.key_value_memory_dict.items():
            assert all(torch.equal(a, b) for a, b in zip(states, mine.key_value_memory_dict[i])), n


@pytest.mark.parametrize("out", [500, 1003])
def test_selection_of_the_int8_heads(dev, out):
    """of the logits of forward, bit for bit"""
    torch.manual_seed(out)
    layer = torch.nn.Linear(256, out, bias=False).half().to(dev)
    for head in (W8A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217)), W4A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217))):
        for batch, beams in ((1, 1), (2, 3)):
            x = torch.randint(-127, 128, (batch, beams, 256), dtype=torch.int8, device=dev)
            scores, done = torch.randn(batch, beams, device=dev), torch.zeros(batch, beams, dtype=torch.bool, device=dev)
            got, want = head.beam_search_step(x, scores, 5, done), ops.beam_search_step(head(x).view(batch, beams, out), scores, 5, done)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            own = torch.full((batch, beams), 0.0217, device=dev)
            scaled = head.beam_search_step(x, scores, 5, x_scale=own)
            assert scaled.tokens.shape == (batch, beams) or scaled.tokens.shape == (batch, 5)
        with pytest.raises(RuntimeError):
            head.beam_search_step(x[0], scores, 5)


def test_heads_without_entries(dev):
    layer = torch.nn.Linear(256, 500, bias=False).half().to(dev)
    scores = torch.zeros(0, 4, device=dev)
    for head in (W8A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217)), W4A8B16O16Linear.from_fp16(layer, torch.tensor(0.0217)), MXFP4Linear.from_fp16(layer)):
        x = torch.zeros(0, 4, 256, dtype=torch.float16 if isinstance(head, MXFP4Linear) else torch.int8, device=dev)
        got = head.beam_search_step(x, scores, 3)
        assert all(t.shape == (0, 3) for t in got)
