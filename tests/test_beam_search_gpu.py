"""Selection over beams and vocabulary against 64 bits.

Scores: the sum of exponentials has terms that are off by less than 6e-11 of themselves (the polynomial's first missing term, r^3 / 6 with r up to ln 2 / 1024) and is held in 64 bits, so a score is
within 1e-9 of what it is in 64 bits (that much of slack for its logarithm and sums), and written with half a step of fp32.  Tokens and parents have to be equal: no two
candidates of different scores in these inputs are nearer than 1e-8, which the reference asserts."""
import numpy as np
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def reference(logits, scores, count, done=None):
    l, own = logits.detach().cpu().double().numpy(), scores.cpu().double().numpy()
    batch, beams, vocab = l.shape
    out = (np.full((batch, count), -np.inf), np.full((batch, count), -1, np.int64), np.full((batch, count), -1, np.int64))
    for b in range(batch):
        offers = []
        for i in range(beams):
            if not np.isfinite(own[b, i]):
                continue
            if done is not None and bool(done[b, i]):
                offers.append((own[b, i], i, 0, -1))
                continue
            row = l[b, i]
            m = row.max()
            if not np.isfinite(m):
                continue
            below, log_sum = row - m, np.log(np.exp(row - m).sum())        # (not m + log_sum: next to -3e38 nothing of the logarithm is left)
            for place, t in enumerate(np.argsort(-row, kind="stable")[:count]):
                if row[t] > -np.inf:
                    offers.append((own[b, i] + (below[t] - log_sum), i, place, int(t)))
        offers.sort(key=lambda o: (-o[0], o[1], o[2]))
        for x, y in zip(offers, offers[1:count + 1]):
            assert x[1] == y[1] or x[0] == y[0] or x[0] - y[0] > 1e-8, "candidates too near each other for this test: other inputs"
        for n, (s, i, _, t) in enumerate(offers[:count]):
            out[0][b, n], out[1][b, n], out[2][b, n] = s, t, i
    return out


def check(logits, scores, count, done=None):
    got = ops.beam_search_step(logits, scores, count, done)
    want = reference(logits, scores, count, done)
    assert got.scores.dtype == torch.float32 and got.tokens.dtype == got.parents.dtype == torch.int64
    assert np.array_equal(got.parents.cpu().numpy(), want[2]) and np.array_equal(got.tokens.cpu().numpy(), want[1])
    s = got.scores.cpu().double().numpy()
    assert np.array_equal(np.isneginf(s), np.isneginf(want[0]))
    fine = np.isfinite(want[0])
    s, w = s[fine], want[0][fine]
    assert np.all(np.abs(s - w) <= np.abs(w) * 2.0 ** -24 + 1e-9 + 2.0 ** -149)
    return got


def make(batch, beams, vocab, dtype, dev, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(1000 * batch + 100 * beams + vocab + seed)
    logits = (spread * torch.randn(batch, beams, vocab, generator=g)).to(TYPES[dtype])
    return logits.to(dev), (-20 + 2 * torch.randn(batch, beams, generator=g)).to(dev)


# one token, fewer than a load's, lanes and batches with a value more or less, cut into segments or not
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("batch,beams,vocab,count", [
    (1, 1, 1, 1), (2, 3, 1, 3), (1, 4, 3, 8), (3, 2, 7, 4), (1, 5, 9, 10), (2, 4, 100, 8), (1, 64, 33, 64), (5, 3, 511, 6), (2, 4, 2047, 8), (1, 3, 2048, 20), (1, 2, 2049, 64),
    (3, 1, 4100, 2), (2, 6, 8193, 17), (1, 4, 50280, 8), (2, 5, 50277, 10), (1, 16, 20000, 32), (40, 8, 1000, 16), (300, 4, 300, 8)])
def test_sizes(dev, dtype, batch, beams, vocab, count):
    check(*make(batch, beams, vocab, dtype, dev), count)


@pytest.mark.parametrize("batch,beams,vocab", [(64, 8, 50280), (600, 3, 9001), (1100, 4, 5000)])
def test_many_rows(dev, batch, beams, vocab):
    """rows in several batches of a workgroup; sampled entries"""
    g = torch.Generator(device=dev).manual_seed(vocab)
    logits = torch.randn(batch, beams, vocab, generator=g, device=dev).mul_(2).bfloat16()
    scores = torch.randn(batch, beams, generator=g, device=dev)
    got = ops.beam_search_step(logits, scores, 2 * beams)
    for b in (0, 1, batch // 2, batch - 1):
        want = reference(logits[b:b + 1], scores[b:b + 1], 2 * beams)
        assert np.array_equal(got.tokens[b:b + 1].cpu().numpy(), want[1]) and np.array_equal(got.parents[b:b + 1].cpu().numpy(), want[2])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [40, 3000, 20001])
def test_masks(dev, dtype, vocab):
    """a part, nearly all, and all of a beam's tokens; the type's lowest value as a mask"""
    logits, scores = make(2, 6, vocab, dtype, dev, spread=3.0)
    g = torch.Generator().manual_seed(vocab)
    logits[0, 1].masked_fill_((torch.rand(vocab, generator=g) < 0.9).to(dev), float("-inf"))
    logits[0, 2, 3:] = float("-inf")
    logits[0, 3] = float("-inf")
    logits[1, 0, 5:] = torch.finfo(logits.dtype).min
    logits[1, 1] = torch.finfo(logits.dtype).min
    logits[1, 2, 1:] = float("-inf")
    check(logits, scores, 12)
    for b in range(2):
        scores[b] = 0
        scores[b, 2 - b] = 50.0                                    # the masked beam above the others
    check(logits, scores, 12)


def test_fewer_candidates_than_places(dev):
    logits, scores = make(3, 4, 9, "fp32", dev)
    logits[0, :, 1:] = float("-inf")
    scores[1, 1:] = float("-inf")
    scores[2] = float("-inf")
    got = check(logits, scores, 20)
    assert int((got.parents[0] >= 0).sum()) == 4 and int((got.parents[1] >= 0).sum()) == 9 and int((got.parents[2] >= 0).sum()) == 0


@pytest.mark.parametrize("vocab", [50, 30000])
def test_beams_that_are_done(dev, vocab):
    logits, scores = make(3, 4, vocab, "fp16", dev)
    done = torch.tensor([[False, True, False, False], [True, True, True, True], [False, False, False, True]], device=dev)
    scores[0, 1], scores[2, 3] = scores[0].max() + 1, float("-inf")
    logits[1] = float("nan")                                       # not read
    logits[0, 1, 0] = float("inf")
    got = check(logits, scores, 8, done)
    assert got.tokens[0, 0] == -1 and got.parents[0, 0] == 1 and got.scores[0, 0] == scores[0, 1]
    assert sorted(got.parents[1, :4].tolist()) == [0, 1, 2, 3] and (got.parents[1, 4:] == -1).all()
    check(logits, scores, 8, done.t().contiguous().t())


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [20, 5000, 40000])
def test_beams_without_a_distribution(dev, dtype, vocab):
    """NaN or +inf anywhere in a row, and scores that are no numbers: nothing is offered, the others stay"""
    for at in (0, vocab // 2, vocab - 1):
        for what in (float("nan"), -float("nan"), float("inf")):
            logits, scores = make(1, 4, vocab, dtype, dev, seed=at)
            logits[0, 2, at] = what
            got = check(logits, scores, 8)
            assert 2 not in got.parents[0].tolist()
    logits, scores = make(1, 4, vocab, dtype, dev)
    scores[0, 0], scores[0, 1] = float("nan"), float("inf")
    got = check(logits, scores, 8)
    assert set(got.parents[0].tolist()) <= {2, 3}


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_equal_candidates(dev, dtype):
    """beams with the same logits and scores, and equal logits: the lower beam, then the lower token"""
    for vocab in (16, 3000, 50280):
        row = torch.zeros(vocab, device=dev)
        row[vocab // 3:] = 1.0
        logits = row.expand(2, 4, vocab).to(TYPES[dtype])
        scores = torch.full((2, 4), -3.0, device=dev)
        got = check(logits.contiguous(), scores, 16)
        assert got.parents[0].tolist() == [0] * min(16, vocab - vocab // 3) + [1] * (16 - min(16, vocab - vocab // 3))
        g = torch.Generator().manual_seed(vocab)
        mixed = torch.randint(0, 4, (vocab,), generator=g).to(TYPES[dtype]).to(dev)
        check(mixed.expand(3, 5, vocab).contiguous(), torch.zeros(3, 5, device=dev), 40)


def test_the_first_step(dev):
    """one beam with 0, the others not there"""
    logits, scores = make(2, 4, 1000, "fp16", dev)
    scores[:, 0], scores[:, 1:] = 0, float("-inf")
    got = check(logits, scores, 8)
    assert not got.parents.any()


@pytest.mark.parametrize("spread", [1e-3, 30.0, 3000.0])
def test_logits_of_any_size(dev, spread):
    for dtype in ("fp16", "fp32"):
        check(*make(2, 3, 4000, dtype, dev, spread=spread), 6)
    logits, scores = make(2, 3, 4000, "fp32", dev, spread=1e30)
    check(logits, scores, 3)
    logits, scores = make(2, 3, 4000, "fp32", dev)
    check(logits + 1e6, scores, 6)
    check(logits - 3e6, scores, 6)


def test_rows_as_they_lie(dev):
    """padded vocabularies, on any address, entries and beams in another order, one row for all beams"""
    base = torch.randn(3, 5, 5001, device=dev).half()
    scores = torch.randn(3, 5, device=dev)
    for logits in (base[..., :5000], base[..., 1:], base[:, 1:4, 7:3000], base[::2], base.transpose(0, 1).contiguous().transpose(0, 1)):
        own = scores[:logits.shape[0], :logits.shape[1]] if logits.shape[0] == 3 else scores[::2]
        got, want = ops.beam_search_step(logits, own, 7), ops.beam_search_step(logits.contiguous(), own.contiguous(), 7)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.parents, want.parents)
        assert (got.scores - want.scores).abs().max() <= 2.0 ** -22 * want.scores.abs().max()
        check(logits, own, 7)
    one = torch.randn(2, 1, 700, device=dev).expand(2, 6, 700)
    check(one, torch.arange(12.0, device=dev).view(2, 6), 9)


def test_no_entries(dev):
    got = ops.beam_search_step(torch.zeros(0, 4, 100, device=dev), torch.zeros(0, 4, device=dev), 8)
    assert [t.shape for t in got] == [(0, 8)] * 3


def test_refusals(dev):
    logits, scores = torch.zeros(2, 4, 100, device=dev), torch.zeros(2, 4, device=dev)
    for args in ((logits[0], scores, 4), (logits.int(), scores, 4), (logits, scores.half(), 4), (logits, scores[:, :3], 4), (logits, scores, 0), (logits, scores, -1),
                 (logits.transpose(1, 2), scores, 4), (logits, scores.cpu(), 4), (logits[:, :, :1], scores, 5), (logits, scores, 4, scores), (logits, scores, 4, (scores > 0)[:1]),
                 (logits, scores, 4, (scores > 0).cpu()), (logits[:, :0], scores[:, :0], 1), (logits.double(), scores, 4)):
        with pytest.raises(RuntimeError):
            ops.beam_search_step(*args)
    with pytest.raises(NotImplementedError):
        ops.beam_search_step(logits, scores, 65)
    with pytest.raises(NotImplementedError):
        ops.beam_search_step(torch.zeros(1, 65, 8, device=dev), torch.zeros(1, 65, device=dev), 4)
    with pytest.raises(TypeError):
        ops.beam_search_step(logits, scores, 4.5)


def test_the_same_every_time(dev):
    """two calls, on two streams, and graphs replayed in turn with eager calls between them"""
    cases = [make(2, 4, 50280, "fp16", dev, seed=s) for s in range(2)]
    first = [ops.beam_search_step(l, s, 8) for l, s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    again = []
    for st, (l, s) in zip(streams, cases):
        with torch.cuda.stream(st):
            again.append(ops.beam_search_step(l, s, 8))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for l, s in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.beam_search_step(l, s, 8))
        graphs.append(graph)
    for a, b in zip(first, again):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for step in range(3):
        for n, (l, s) in enumerate(cases):
            fresh = make(2, 4, 50280, "fp16", dev, seed=10 * step + n + 5)
            l.copy_(fresh[0])
            s.copy_(fresh[1])
        want = [ops.beam_search_step(l, s, 8) for l, s in cases]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), step


def far_and_equal(dev, vocab, seed):
    """8 beams, all of them with the logits and the score of the first but for one whose logits are far from 0"""
    logits, scores = make(1, 1, vocab, "fp32", dev, seed)
    logits, scores = logits.expand(1, 8, vocab).clone(), scores.expand(1, 8).clone()
    logits[0, 1] += 3e6
    scores[0, 1] = -1e6
    return logits, scores


@pytest.mark.parametrize("vocab", [30000, 100000])
def test_a_beam_does_not_see_the_others(dev, vocab):
    """equal beams stay equal to the last bit, whichever beams share a wave with them"""
    for seed in range(12):
        got = ops.beam_search_step(*far_and_equal(dev, vocab, seed), 35)
        want = [0, 2, 3, 4, 5, 6, 7] * 5
        assert got.parents[0].tolist() == want, seed
        assert all(len(set(got.tokens[0, 7 * i:7 * i + 7].tolist())) == 1 for i in range(5)), seed


def test_workspace_that_held_other_things(dev):
    """parts of beams that are done are not written, and nothing comes of what lay there"""
    logits, scores = make(2, 7, 40000, "fp16", dev)
    done = torch.tensor([[False, True, False, False, True, False, False], [True, False, True, False, False, False, True]], device=dev)
    outs = []
    for byte in (0, 0x7f, 0xff, 0xc1):
        held = [torch.full((n,), byte, dtype=torch.uint8, device=dev) for n in (1 << 12, 1 << 16, 1 << 18, 1 << 20) for _ in range(2)]
        torch.cuda.synchronize()
        del held
        outs.append(check(logits, scores, 9, done))
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, outs[0]))


@pytest.mark.parametrize("batch,beams,vocab,count,dtype", [
    (1, 1, 1 << 20, 64, "fp32"), (1, 1, 1 << 20, 7, "fp16"), (1, 3, (1 << 20) - 5, 20, "bf16"), (1, 64, 50280, 64, "fp32"), (2, 64, 30011, 33, "fp16"), (1, 40, 5000, 1, "fp32"),
    (130, 2, 9000, 64, "fp32"), (1, 2, 256000, 48, "fp32")])
def test_long_rows_and_many_lists(dev, batch, beams, vocab, count, dtype):
    g = torch.Generator().manual_seed(vocab + count)
    # (values that are all different, of one type: no two candidates of a beam are equal, and the scores of beams differ by what no logits do)
    logits = torch.stack([torch.randperm(vocab, generator=g) for _ in range(min(batch * beams, 4))]).repeat(-(-batch * beams // 4), 1)[:batch * beams].float()
    logits = (logits.view(batch, beams, vocab) * (12.0 / vocab)).to(TYPES[dtype]).to(dev)
    scores = (torch.arange(batch * beams).view(batch, beams) * 0.0137 - 5).to(dev)
    check(logits, scores, count)


@pytest.mark.parametrize("rows", [(3, 4), (20, 8)])
def test_captured_and_on_another_stream(dev, rows):
    """two graphs with workspaces of their own, replayed in turn with eager calls between them"""
    inputs = [make(*rows, 30000, "bf16", dev, seed) for seed in range(2)]
    ops.beam_search_step(*inputs[0], 8)
    graphs, outs = [], []
    for logits, scores in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.beam_search_step(logits, scores, 8))
        graphs.append(graph)
    for step in range(3):
        for i, (logits, scores) in enumerate(inputs):
            new = make(*rows, 30000, "bf16", dev, 10 * step + i)
            logits.copy_(new[0])
            scores.copy_(new[1])
        want = [ops.beam_search_step(*x, 8) for x in inputs]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w)), step
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.beam_search_step(*inputs[0], 8)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))


def test_offsets_past_32_bits(dev):
    """rows more than 4 GiB into the logits"""
    batch, vocab = 2100, 1 << 20
    logits = torch.full((batch, 1, vocab), -30.0, dtype=torch.float16, device=dev)
    some = [0, 1023, 1024, 2047, 2048, batch - 1]
    for i, b in enumerate(some):
        logits[b, 0, 100 * i + 7], logits[b, 0, vocab - 1 - i] = 5.0, 4.0
    got = ops.beam_search_step(logits, torch.zeros(batch, 1, device=dev), 2)
    for i, b in enumerate(some):
        assert got.tokens[b].tolist() == [100 * i + 7, vocab - 1 - i]


@pytest.mark.parametrize("batch,beams,vocab,count", [(1, 24, 40000, 64), (2, 30, 70001, 60), (1, 64, 20000, 33)])
def test_many_beams(dev, batch, beams, vocab, count):
    """equal logits, one beam above all others, half of the beams done or not there"""
    g = torch.Generator().manual_seed(vocab)
    mixed = torch.randint(0, 5, (vocab,), generator=g).half().to(dev).expand(batch, beams, vocab).contiguous()
    check(mixed, torch.zeros(batch, beams, device=dev), count)
    logits, scores = make(batch, beams, vocab, "fp32", dev)
    scores = torch.linspace(-40, -30, beams, device=dev).expand(batch, beams).clone()
    scores[:, beams // 2] = 25.0
    check(logits, scores, count)
    scores[:, beams // 2] = -31.7
    scores[:, ::3] = float("-inf")
    done = torch.zeros(batch, beams, dtype=torch.bool, device=dev)
    done[:, 1::4] = True
    check(logits, scores, count, done)
    check(logits, scores, 1, done)
