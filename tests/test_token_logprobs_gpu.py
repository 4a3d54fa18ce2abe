"""Log probabilities, entropies and best alternatives of logits against 64 bits.

The kernel works in fp32, unit 2^-24.  The sum of exponentials is, in a lane, a chain of a 256th of the vocabulary, raised to a larger
maximum at most once in 16 of its terms, then some 20 joins; each exponential is within 3 units and 1.5 |d| (d = l - m, the rounding
of its argument), which with its weight e^d is below 1.  So ln s is within V/200 + 64 units; the difference in front of it and the last one add
their own roundings, at most 4 units of what they are between.  The entropy's second term, t / s, has the same share of itself."""
import numpy as np
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def reference(logits, tokens, top):
    """(logprobs, entropy, top logprobs, top tokens, ln s) in 64 bits, the order of equal logits by index"""
    l = logits.detach().cpu().double().numpy()
    t = tokens.cpu().numpy()
    m = l.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        e = np.exp(l - m)
        s = e.sum(-1, keepdims=True)
        lse = m + np.log(s)
        d = np.where(e > 0, l - m, 0.0)
        entropy = (np.log(s) - (e * d).sum(-1, keepdims=True) / s)[:, 0]
        lp = np.where(t < 0, 0.0, np.take_along_axis(l, np.clip(t, 0, l.shape[1] - 1)[:, None], 1)[:, 0] - lse[:, 0])
    at = np.argsort(-l, axis=-1, kind="stable")[:, :top]
    return lp, entropy, np.take_along_axis(l, at, 1) - lse, at, np.log(s)[:, 0]


def check(got, logits, tokens, top, extra=0.0):
    """extra: what the logits themselves may be off by"""
    lp, h, best, at, ln_s = reference(logits, tokens, top)
    V = logits.shape[-1]
    chain = (V / 200 + 64) * U + 2 * extra
    g = [t.cpu().double().numpy() for t in got]
    with np.errstate(invalid="ignore"):
        for a, b in ((g[0], lp), (g[2], best)):
            assert np.array_equal(np.isneginf(a), np.isneginf(b)) and np.array_equal(np.isnan(a), np.isnan(b))
            fine = np.isfinite(b)
            off = np.abs(a - b)[fine]
            bound = (chain + 4 * U * (1 + np.abs(b) + np.broadcast_to(ln_s[:, None] if b.ndim > 1 else ln_s, b.shape)))[fine]
            assert np.all(off <= bound), (off / bound).max()
        fine = np.isfinite(h)
        assert np.array_equal(np.isnan(g[1]), ~fine)
        assert np.all(np.abs(g[1] - h)[fine] <= (chain * (1 + h - ln_s) + 4 * U * (1 + h + ln_s))[fine])
    assert np.array_equal(got.top_tokens.cpu().numpy(), at)


def make(rows, vocab, dtype, dev, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(7 * rows + vocab + seed)
    logits = (spread * torch.randn(rows, vocab, generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    return logits.to(dev), tokens.to(dev)


# one value, fewer than a load's, lanes and batches with a value more or less, cut into segments or not
VOCABS = [1, 2, 7, 8, 9, 63, 64, 513, 2047, 2048, 8191, 8192, 8193, 16390, 50280]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", TYPES)
def test_vocabularies(dev, vocab, dtype):
    for rows, top in ((1, min(vocab, 5)), (6, 0), (3, min(vocab, 64))):
        logits, tokens = make(rows, vocab, TYPES[dtype], dev)
        check(ops.token_logprobs(logits, tokens, top=top), logits, tokens, top)


@pytest.mark.parametrize("rows,vocab", [(256, 7), (257, 64), (1000, 513), (300, 2048), (301, 2049), (259, 4096), (258, 4097), (4097, 2500), (4096, 9001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dev, dtype, rows, vocab):
    """Rows of a wave each; the last workgroup has fewer of them than waves."""
    for top in (0, min(vocab, 6), min(vocab, 64)):
        logits, tokens = make(rows, vocab, TYPES[dtype], dev)
        logits[5] = float("-inf")
        logits[5, vocab // 2] = 1.0
        check(ops.token_logprobs(logits, tokens, top=top), logits, tokens, top)


@pytest.mark.parametrize("top", [0, 1, 2, 5, 20, 63, 64])
@pytest.mark.parametrize("rows", [1, 40, 1500])
def test_numbers_of_alternatives(dev, top, rows):
    logits, tokens = make(rows, 10007, torch.bfloat16, dev)       # (many equal values)
    check(ops.token_logprobs(logits, tokens, top=top), logits, tokens, top)


@pytest.mark.parametrize("dtype,vocab", [("bf16", 256000), ("fp32", 256003), ("fp16", 131072)])
@pytest.mark.parametrize("rows", [1, 5])
def test_large_vocabularies(dev, dtype, vocab, rows):
    logits, tokens = make(rows, vocab, TYPES[dtype], dev)
    check(ops.token_logprobs(logits, tokens, top=3), logits, tokens, 3)


@pytest.mark.parametrize("shape", ["rising", "falling", "equal", "one hot", "two values"])
@pytest.mark.parametrize("rows", [1, 700, 4100])
def test_orders_of_the_values(dev, shape, rows):
    V = 20011 if rows < 1000 else 5003
    row = {"rising": torch.linspace(-9, 9, V), "falling": torch.linspace(9, -9, V), "equal": torch.full((V,), 1.25),
           "one hot": torch.zeros(V).index_fill_(0, torch.tensor([V - 1]), 80.0), "two values": (torch.arange(V) % 3 == 1).float()}[shape]
    logits = row.repeat(rows, 1).to(dev)
    tokens = torch.arange(rows, device=dev) * 13 % V
    check(ops.token_logprobs(logits, tokens, top=17), logits, tokens, 17)


@pytest.mark.parametrize("dtype,vocab", [("fp16", 16387), ("bf16", 16391), ("fp32", 8195), ("fp16", 24581), ("fp32", 12291)])
@pytest.mark.parametrize("rows", [512, 700, 1030])
def test_values_behind_the_last_whole_load(dev, dtype, vocab, rows):
    """They are all that is left for the last segment; the best value among them, or none that counts, or only NaNs."""
    logits, tokens = make(rows, vocab, TYPES[dtype], dev)
    logits[1::3, -1] = 30.0
    logits[2::3, -3:] = float("-inf")
    check(ops.token_logprobs(logits, tokens, top=5), logits, tokens, 5)
    logits[0, -3:] = float("nan")
    got = ops.token_logprobs(logits, tokens, top=5)
    assert torch.isnan(got.entropy[0]) and ((got.top_tokens >= 0) & (got.top_tokens < vocab)).all()


@pytest.mark.parametrize("rows", [2, 600, 4100])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(dev, dtype, rows):
    """-inf and the type's lowest value in masked places, given tokens among them; fewer values left than alternatives asked for."""
    V = 9001 if rows < 1000 else 3001
    for fill in (float("-inf"), torch.finfo(TYPES[dtype]).min):
        logits, tokens = make(rows, V, TYPES[dtype], dev)
        hidden = torch.rand(rows, V, generator=torch.Generator().manual_seed(3)) < 0.5
        hidden[0] = True
        hidden[0, [4, 2000, V - 2]] = False
        logits.masked_fill_(hidden.to(dev), fill)
        tokens[0] = 7
        check(ops.token_logprobs(logits, tokens, top=6), logits, tokens, 6)
    logits = torch.full((rows, V), torch.finfo(TYPES[dtype]).min, dtype=TYPES[dtype], device=dev)       # nothing but the lowest value: all the same
    tokens = torch.zeros(rows, dtype=torch.int64, device=dev)
    got = ops.token_logprobs(logits, tokens, top=2)
    assert torch.allclose(got.logprobs, torch.full_like(got.logprobs, -np.log(V)), rtol=1e-6) and (got.top_tokens == torch.tensor([0, 1], device=dev)).all()


@pytest.mark.parametrize("vocab", [9, 2500])
@pytest.mark.parametrize("rows", [1, 300, 4100])
def test_certain_tokens(dev, rows, vocab):
    """All of the weight on one token: its log probability and the entropy are 0 to within the bounds, and on the right side of it"""
    g = torch.Generator().manual_seed(rows + vocab)
    logits, tokens = torch.full((rows, vocab), -3e4), torch.randint(0, vocab, (rows,), generator=g)
    logits[torch.arange(rows), tokens] = 20 * torch.randn(rows, generator=g)
    logits, tokens = logits.to(dev), tokens.to(dev)
    got = ops.token_logprobs(logits, tokens, 2)
    check(got, logits, tokens, 2)
    assert (got.logprobs <= 0).all() and (got.top_logprobs <= 0).all() and (got.entropy >= 0).all()


@pytest.mark.parametrize("vocab", [5, 3000, 50280])
@pytest.mark.parametrize("rows", [4, 900, 4100])
def test_rows_without_a_distribution(dev, vocab, rows):
    """All masked, a NaN, an infinity: NaN in that row alone, and indices that lie in the row."""
    logits, tokens = make(rows, vocab, torch.float32, dev)
    clean = ops.token_logprobs(logits, tokens, top=3)
    logits[0] = float("-inf")
    logits[1, vocab // 2] = float("nan")
    logits[2, vocab - 1] = float("inf")
    got = ops.token_logprobs(logits, tokens, top=3)
    assert torch.isnan(got.logprobs[:3]).all() and torch.isnan(got.entropy[:3]).all() and torch.isnan(got.top_logprobs[:3]).all()
    assert ((got.top_tokens >= 0) & (got.top_tokens < vocab)).all()
    assert all(torch.equal(a[3:], b[3:]) for a, b in zip(got, clean))
    tokens[:3] = -1
    assert (ops.token_logprobs(logits, tokens).logprobs[:3] == 0).all()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,vocab", [(7, 300), (3, 50280), (2000, 50)])
def test_tokens_outside_the_vocabulary(dev, dtype, rows, vocab):
    logits, tokens = make(rows, vocab, torch.float16, dev)
    tokens = tokens.to(dtype)
    want = ops.token_logprobs(logits, tokens).logprobs
    ends = [-1, -100, vocab, torch.iinfo(dtype).max, torch.iinfo(dtype).min]
    if dtype == torch.int64:
        ends += [1 << 32, -(1 << 32)]                              # (their low words are 0)
    for bad in ends:
        t = tokens.clone()
        t[1] = bad
        got = ops.token_logprobs(logits, t)
        assert got.logprobs[1] == 0 if bad < 0 else torch.isnan(got.logprobs[1])
        keep = torch.arange(rows, device=dev) != 1
        assert torch.equal(got.logprobs[keep], want[keep]) and torch.isfinite(got.entropy).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_padded_logits(dev, dtype):
    """Rows apart from each other and off every boundary; dimensions in front."""
    for vocab, pad, shift in ((50280, 8, 0), (1000, 3, 1), (1003, 0, 0), (777, 20, 5)):
        logits, tokens = make(4, vocab, TYPES[dtype], dev)
        wide = torch.full((4, vocab + pad + shift), 99.0, dtype=logits.dtype, device=dev)
        wide[:, shift:shift + vocab] = logits
        check(ops.token_logprobs(wide[:, shift:shift + vocab], tokens, top=4), logits, tokens, 4)
    logits, tokens = make(6, 500, TYPES[dtype], dev)
    flat = ops.token_logprobs(logits, tokens, top=2)
    got = ops.token_logprobs(logits.view(2, 3, 500), tokens.view(2, 3), top=2)
    assert got.logprobs.shape == (2, 3) and got.top_tokens.shape == (2, 3, 2)
    assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, flat))
    # every position but the last of each sequence (a copy is made), of one sequence (none is)
    shifted = ops.token_logprobs(logits.view(2, 3, 500)[:, :-1], tokens.view(2, 3)[:, 1:])
    assert torch.equal(shifted.entropy, flat.entropy.view(2, 3)[:, :-1])
    one = ops.token_logprobs(logits[0], tokens[0], top=1)
    assert one.logprobs.shape == () and one.top_tokens.shape == (1,) and torch.equal(one.logprobs, flat.logprobs[0])
    empty = ops.token_logprobs(logits[:0], tokens[:0], top=2)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 2)


def test_rows_beyond_32_bits(dev):
    """The last rows lie further than 2^31 values behind the first."""
    vocab, rows = 50280, 3
    store = torch.empty((1 << 31) + 3 * vocab, dtype=torch.bfloat16, device=dev)
    logits = store.as_strided((rows, vocab), ((1 << 30) + 8, 1))
    fresh, tokens = make(rows, vocab, torch.bfloat16, dev)
    logits.copy_(fresh)
    check(ops.token_logprobs(logits, tokens, top=3), fresh, tokens, 3)


def test_the_same_bits_again(dev):
    """No sum depends on the order in which workgroups end."""
    for rows in (1, 300, 4099):
        logits, tokens = make(rows, 50280, torch.float16, dev)
        want = ops.token_logprobs(logits, tokens, top=5)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(logits, tokens, top=5), want))


def test_on_another_stream_and_replayed(dev):
    logits, tokens = make(3, 50280, torch.float16, dev)
    want = ops.token_logprobs(logits, tokens, top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.token_logprobs(logits, tokens, top=5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                             # (each with a workspace of its own)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.token_logprobs(logits, tokens, top=5)))
    for i in range(3):
        logits.copy_(torch.randn(3, 50280, device=dev))
        tokens.random_(0, 50280)
        for graph, _ in graphs:
            graph.replay()
        now = ops.token_logprobs(logits, tokens, top=5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for _, held in graphs for a, b in zip(held, now)), i


def test_refusals(dev):
    logits, tokens = make(4, 300, torch.float16, dev)
    for bad in (dict(tokens=tokens[:3]), dict(tokens=tokens.float()), dict(tokens=tokens.cpu()), dict(logits=logits.cpu()), dict(top=301), dict(top=-1),
                dict(logits=logits.to(torch.int8)), dict(logits=logits.double()), dict(logits=logits[:, :0])):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(**{"logits": logits, "tokens": tokens, **bad})
    with pytest.raises(NotImplementedError):
        ops.token_logprobs(logits, tokens, top=65)


def test_answers_are_tensors_of_their_own(dev):
    """Some lie in one allocation, and none of them notices: writing one leaves the others, copies and files hold what they should."""
    import copy
    import io
    logits, tokens = make(6, 300, torch.float16, dev)
    got = ops.token_logprobs(logits, tokens, top=3)
    want = [t.clone() for t in got]
    assert [t.dtype for t in got] == [torch.float32, torch.float32, torch.float32, torch.int64] and all(t.is_contiguous() and not t.requires_grad for t in got)
    for i, t in enumerate(got):
        t.zero_()
        assert (t == 0).all() and all(torch.equal(a, b) for a, b in zip(got[i + 1:], want[i + 1:]))
    again = ops.token_logprobs(logits, tokens, top=3)
    file = io.BytesIO()
    torch.save(list(again), file)
    file.seek(0)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(again, torch.load(file, weights_only=True), copy.deepcopy(list(again))))
    # usable as a leaf and in a graph of gradients
    leaf = again.logprobs.requires_grad_()
    (2 * leaf).sum().backward()
    assert (leaf.grad == 2).all()


def test_in_inference_mode(dev):
    logits, tokens = make(6, 300, torch.float16, dev)
    want = ops.token_logprobs(logits, tokens, top=3)
    with torch.inference_mode():
        got = ops.token_logprobs(logits.clone(), tokens, top=3)
        got.logprobs.add_(1).sub_(1)
    assert all(t.is_inference() for t in got) and not any(t.is_inference() for t in want)
    assert torch.equal(got.entropy, want.entropy) and torch.equal(got.top_tokens, want.top_tokens)
