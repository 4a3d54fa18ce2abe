"""Log probabilities of rows that are masked with a large finite number, and of logits that are large themselves, against 64 bits.

The bounds are those of test_token_logprobs_gpu.check with 32 units (2^-24) more in the logarithm of the sum, for any way a row is cut: a lane
adds at most 32 terms of a batch one after the other, at most V/1024 batches of at most 5 units each (the sum, and a raised maximum),
then some 16 joins; an exponential is within 3 units and 2.2 |d| of them (a difference and a product, each rounded, and the rounding of log2 e), and the mean
of |d| over the distribution is at most ln V, 12.5.  V/205 + 32 + 16 + 3 + 28 units are within V/200 + 64 + 32."""
import pytest
import torch

from quamba_amd import ops
from test_token_logprobs_gpu import TYPES, U, make
from test_token_logprobs_gpu import check as check_near_zero

pytestmark = pytest.mark.gpu
MORE = 16 * U                              # (counted twice by check)
FILLS = [-6e4, -1e6, -1.1e6, -1e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e32, -1e37]


def check(got, logits, tokens, top, extra=MORE):
    """As seen from each row's largest logit, where nothing asked for is another: 64 bits do not hold -1e30 and the logarithm of a sum beside it."""
    wide = logits.double()
    check_near_zero(got, wide - wide.amax(-1, keepdim=True), tokens, top, extra)


def _vocab(rows):
    return {1: 50283, 64: 20011, 600: 5003, 4100: 3001}[rows]


@pytest.mark.parametrize("rows", [1, 64, 600, 4100])
@pytest.mark.parametrize("dtype,fill", [("fp16", -6e4)] + [(t, f) for t in ("bf16", "fp32") for f in FILLS])
def test_masked_with_a_finite_number(dev, dtype, fill, rows):
    """Half of the vocabulary, and all but three tokens of it (fewer than the alternatives asked for, and a masked token asked for)"""
    V = _vocab(rows)
    for top in (0, 6):
        logits, tokens = make(rows, V, TYPES[dtype], dev)
        hidden = torch.rand(rows, V, generator=torch.Generator().manual_seed(3)) < 0.5
        hidden[0] = True
        hidden[0, [4, 2000, V - 2]] = False
        tokens[0] = 7
        check(ops.token_logprobs(logits.masked_fill(hidden.to(dev), fill), tokens, top=top), logits.masked_fill(hidden.to(dev), fill), tokens, top)
        few = logits.new_full((rows, V), fill)
        for i, at in enumerate((0, V // 2, V - 1)):
            few[:, at] = logits[:, i]
        tokens[::2] = V // 2
        check(ops.token_logprobs(few, tokens, top=top), few, tokens, top)


@pytest.mark.parametrize("rows", [1, 64, 600, 4100])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("fill", [-1e9, -1e30])
def test_whole_parts_of_a_row_masked(dev, dtype, fill, rows):
    """Segments, batches and lanes that hold nothing but the fill: the tokens left are the first, or the last, of the row; none is left"""
    V = _vocab(rows)
    for left in (slice(0, 5), slice(V - 5, V)):
        logits = torch.full((rows, V), fill, dtype=TYPES[dtype], device=dev)
        logits[:, left] = make(rows, 5, TYPES[dtype], dev)[0]
        tokens = torch.full((rows,), left.start + 1, device=dev)
        check(ops.token_logprobs(logits, tokens, top=4), logits, tokens, 4)
    logits = torch.full((rows, V), fill, dtype=TYPES[dtype], device=dev)
    check(ops.token_logprobs(logits, tokens, top=4), logits, tokens, 4)


@pytest.mark.parametrize("rows", [1, 600, 4100])
@pytest.mark.parametrize("offset", [2.0 ** 19, 2.0 ** 21, -3e7, 1e9, -1e10])
def test_logits_far_from_zero(dev, offset, rows):
    """fp32 logits around a large number, as far apart as fp32 can tell them there"""
    V = _vocab(rows)
    logits, tokens = make(rows, V, torch.float32, dev, spread=4.0)
    step = max(1.0, abs(offset) * 2.0 ** -23)
    logits = (logits * step + offset).float()
    check(ops.token_logprobs(logits, tokens, top=3), logits, tokens, 3)


def test_a_nan_among_masked_logits(dev):
    """A NaN still takes its row, and an infinity, whatever the others are masked with"""
    for fill in (-1e10, -1e30, float("-inf")):
        logits = torch.full((3, 9001), fill, device=dev)
        logits[:, 100] = 1.0
        logits[0, 5] = float("nan")
        logits[1, 6] = float("inf")
        got = ops.token_logprobs(logits, torch.full((3,), 100, device=dev), top=2)
        assert torch.isnan(got.logprobs[:2]).all() and torch.isnan(got.entropy[:2]).all()
        assert got.logprobs[2] == 0 and got.entropy[2] == 0 and got.top_tokens[2, 0] == 100
