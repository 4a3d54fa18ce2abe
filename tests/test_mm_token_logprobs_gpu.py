"""Log probabilities of the head's int8 product: against 64 bits, and its best column against the same fp32 logits.

A logit is two products in fp32 of a whole number below 2^24 and two scales: within 2^-23 of itself (the same product elementwise gives
the same bits).  The statistics' bounds are those of the logits' own operator."""
import pytest
import torch

from quamba_amd import ops
from test_token_logprobs_gpu import check as check_logprobs

pytestmark = pytest.mark.gpu


def make(rows, vocab, k, dev, row_scales=True, channel_scales=True, seed=0, pad=None, size=2.5):
    g = torch.Generator().manual_seed(rows + 3 * vocab + 5 * k + seed)
    n = (vocab + 15) // 16 * 16 if pad is None else vocab + pad
    a = torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    unit = size / (74 * 74 * k ** 0.5)                             # (codes of all values have a root mean square of 74)
    a_s = (0.7 + 0.6 * torch.rand(rows if row_scales else 1, generator=g))
    w_s = (0.7 + 0.6 * torch.rand(n if channel_scales else 1, generator=g)) * unit
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    return dict(a=a.to(dev), b=w.to(dev).t(), a_scales=a_s.to(dev), b_scales=w_s.to(dev), tokens=tokens.to(dev))


def logits_of(c, vocab):
    """The logits in fp32, in the kernel's own order of products"""
    acc = (c["a"].cpu().double() @ c["b"].cpu().double()[:, :vocab]).float()
    s = c["b_scales"].cpu()
    return c["a_scales"].cpu()[:, None] * ((s if s.numel() == 1 else s[:vocab]) * acc)


def check(got, c, vocab, top=0):
    logits = logits_of(c, vocab)
    check_logprobs(got, logits, c["tokens"], top, extra=0.0)


# rows and columns around every tile's edge, K of one 16-byte piece, less and more than a tile's depth
@pytest.mark.parametrize("rows", [1, 2, 16, 33, 63, 64, 65, 128, 129, 200, 256, 257, 600])
@pytest.mark.parametrize("vocab,k", [(1000, 256), (50, 16), (777, 144)])
def test_rows(dev, rows, vocab, k):
    c = make(rows, vocab, k, dev)
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("vocab", [1, 2, 15, 16, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 5001])
@pytest.mark.parametrize("rows", [3, 100, 300])
def test_vocabularies(dev, rows, vocab):
    c = make(rows, vocab, 384, dev)
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("k", [16, 112, 128, 240, 256, 272, 384, 400, 512, 768, 1040, 2560, 4096])
@pytest.mark.parametrize("rows", [4, 90, 270])
def test_depths(dev, rows, k):
    c = make(rows, 600, k, dev)
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=600), c, 600, 1)


@pytest.mark.parametrize("rows", [5, 130, 300])
@pytest.mark.parametrize("row_scales", [True, False])
@pytest.mark.parametrize("channel_scales", [True, False])
def test_scales(dev, rows, row_scales, channel_scales):
    c = make(rows, 900, 512, dev, row_scales, channel_scales)
    check(ops.scaled_mm_token_logprobs(**c, vocab=900), c, 900)


@pytest.mark.parametrize("rows,vocab,k", [(1, 50280, 768), (64, 50280, 256), (1021, 50277, 128), (2, 256000, 64)])
def test_whole_heads(dev, rows, vocab, k):
    c = make(rows, vocab, k, dev)
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("rows", [6, 300])
def test_certain_tokens(dev, rows):
    """Logits so far apart that most rows have all of their weight on one token: on the right side of 0"""
    c = make(rows, 500, 256, dev, size=3000.0)
    c["tokens"] = logits_of(c, 500).argmax(-1).to(dev)
    got = ops.scaled_mm_token_logprobs(**c, top=1, vocab=500)
    check(got, c, 500, 1)
    assert (got.logprobs <= 0).all() and (got.top_logprobs <= 0).all() and (got.entropy >= 0).all()


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_columns_behind_the_vocabulary_count_for_nothing(dev, rows):
    c = make(rows, 500, 256, dev, pad=300)
    want = ops.scaled_mm_token_logprobs(**c, top=1, vocab=500)
    check(want, c, 500, 1)
    c["b"][:, 500:] = 127
    c["b_scales"][500:] = float("inf")
    got = ops.scaled_mm_token_logprobs(**c, top=1, vocab=500)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    c = make(rows, 512, 256, dev, pad=0)
    assert all(torch.equal(x, y) for x, y in zip(ops.scaled_mm_token_logprobs(**c, top=1), ops.scaled_mm_token_logprobs(**c, top=1, vocab=512)))


@pytest.mark.parametrize("rows", [4, 80, 300])
def test_equal_columns_and_large_logits(dev, rows):
    """The lowest index of equal logits, wherever the columns lie; logits far above 88."""
    c = make(rows, 1500, 256, dev, channel_scales=False, size=2000.0)
    c["b"][:, 1400] = c["b"][:, 3]
    c["b"][:, 700] = c["b"][:, 3]
    c["a"][:] = c["b"][:, 3]                                       # column 3 is the best one by far
    got = ops.scaled_mm_token_logprobs(**c, top=1)
    assert (got.top_tokens == 3).all()
    check(got, c, c["b"].shape[1], 1)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows", [6, 100, 300])
def test_tokens_outside_the_vocabulary(dev, dtype, rows):
    c = make(rows, 500, 128, dev)
    c["tokens"] = c["tokens"].to(dtype)
    want = ops.scaled_mm_token_logprobs(**c, vocab=500).logprobs
    ends = [-1, -100, 500, 505, torch.iinfo(dtype).max, torch.iinfo(dtype).min]
    if dtype == torch.int64:
        ends += [1 << 32, (1 << 32) + 3, -(1 << 32)]               # (their low words are columns)
    keep = torch.arange(rows, device=dev) != 1
    for bad in ends:
        c["tokens"] = c["tokens"].clone()
        c["tokens"][1] = bad
        got = ops.scaled_mm_token_logprobs(**c, vocab=500).logprobs
        assert got[1] == 0 if bad < 0 else torch.isnan(got[1])
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("rows", [4, 90, 300])
def test_a_row_whose_scale_is_nan(dev, rows):
    """as the norm leaves it for a row with a NaN: NaN in that row alone, a column that exists"""
    c = make(rows, 700, 128, dev)
    want = ops.scaled_mm_token_logprobs(**c, top=1, vocab=700)
    c["a_scales"][2] = float("nan")
    got = ops.scaled_mm_token_logprobs(**c, top=1, vocab=700)
    assert torch.isnan(got.logprobs[2]) and torch.isnan(got.entropy[2]) and torch.isnan(got.top_logprobs[2, 0]) and 0 <= got.top_tokens[2, 0] < 700
    keep = torch.arange(rows, device=dev) != 2
    assert all(torch.equal(x[keep], y[keep]) for x, y in zip(got, want))


def test_rows_that_lie_apart(dev):
    c = make(70, 300, 256, dev)
    want = ops.scaled_mm_token_logprobs(**c, top=1, vocab=300)
    a, w = torch.full((70, 320), 77, dtype=torch.int8, device=dev), torch.full((304, 288), 77, dtype=torch.int8, device=dev)
    a[:, 16:272], w[:, :256] = c["a"], c["b"].t()
    got = ops.scaled_mm_token_logprobs(**{**c, "a": a[:, 16:272], "b": w[:, :256].t()}, top=1, vocab=300)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("rows,vocab", [(2, 70000), (70000, 130)])
def test_operands_beyond_32_bits(dev, rows, vocab):
    """Rows 32 KiB apart: the last ones lie more than 2^31 bytes behind the first."""
    pitch, k = 32768, 64
    c = make(rows, vocab, k, dev)
    want = ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab)
    large = "a" if rows > vocab else "b"
    n = max(rows, c["b"].shape[1]) if large == "b" else rows
    store = torch.empty(n * pitch, dtype=torch.int8, device=dev)
    rows_apart = store.view(n, pitch)[:, :k]
    rows_apart.copy_(c["a"] if large == "a" else c["b"].t())
    got = ops.scaled_mm_token_logprobs(**{**c, large: rows_apart if large == "a" else rows_apart.t()}, top=1, vocab=vocab)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    few = min(rows, 300)
    part = {k_: (v[:few] if k_ in ("a", "tokens") or (k_ == "a_scales" and v.numel() > 1) else v) for k_, v in c.items()}
    check(ops.TokenLogprobs(*(t[:few] for t in got)), part, vocab, 1)


def test_the_same_bits_again_and_no_rows(dev):
    c = make(300, 2000, 256, dev)
    want = ops.scaled_mm_token_logprobs(**c, top=1)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(ops.scaled_mm_token_logprobs(**c, top=1), want))
    none = ops.scaled_mm_token_logprobs(c["a"][:0], c["b"], c["a_scales"][:1], c["b_scales"], c["tokens"][:0], top=1)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 1)


@pytest.mark.parametrize("rows", [1, 64, 300])
def test_on_another_stream_and_replayed(dev, rows):
    c = make(rows, 5000, 512, dev)
    want = ops.scaled_mm_token_logprobs(**c, top=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.scaled_mm_token_logprobs(**c, top=1)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.scaled_mm_token_logprobs(**c, top=1)))
    for i in range(3):
        c["a"].random_(-127, 128)
        c["tokens"].random_(0, 5000)
        for graph, _ in graphs:
            graph.replay()
        now = ops.scaled_mm_token_logprobs(**c, top=1)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for _, held in graphs for x, y in zip(held, now)), i


def test_refusals(dev):
    c = make(5, 300, 128, dev)
    a, b = c["a"], c["b"]
    for bad in (dict(a=a.float()), dict(a=a[:, :120], b=b[:120]), dict(b=b.contiguous()), dict(a_scales=c["a_scales"][:3]), dict(b_scales=c["b_scales"][:300]),
                dict(a_scales=c["a_scales"].double()), dict(tokens=c["tokens"][:4]), dict(tokens=c["tokens"].to(torch.int16)), dict(vocab=305), dict(vocab=0),
                dict(a=a.cpu()), dict(b=b.cpu()), dict(a=a[:, :64])):
        with pytest.raises(RuntimeError):
            ops.scaled_mm_token_logprobs(**{**c, **bad})
    with pytest.raises(NotImplementedError):
        ops.scaled_mm_token_logprobs(**c, top=2)
