"""Scales of the head's int8 product that are negative, zero, infinite, no number or very large: wherever the column lies, whole tiles and
ragged ones alike.  The logits are the fp32 products a_scale * (b_scale * sum), as the reference of test_mm_token_logprobs_gpu forms them."""
import pytest
import torch

from quamba_amd import ops
from test_finite_masks_gpu import check as check_logprobs
from test_mm_token_logprobs_gpu import logits_of, make

pytestmark = pytest.mark.gpu
ROWS = [1, 4, 64, 70, 128, 300]


def check(got, c, vocab, top):
    check_logprobs(got, logits_of(c, vocab), c["tokens"], top)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab", [700, 2000])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_a_column_whose_scale_is_no_number(dev, rows, vocab, scale):
    """The logit of that column is a NaN in every row (an infinity times 0 is one too), so no row has a distribution"""
    for at in (0, 5, 69, vocab // 2, vocab - 2, vocab - 1):
        c = make(rows, vocab, 128, dev)
        c["b"][:, at] = 0
        c["b_scales"][at] = scale
        got = ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab)
        assert all(torch.isnan(t).all() for t in got[:3]), at
        assert ((got.top_tokens >= 0) & (got.top_tokens < vocab)).all()
        c["b_scales"][at] = 1.0
        check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab", [700, 2000])
def test_a_column_of_minus_infinity(dev, rows, vocab):
    """An infinite scale and a negative sum: masked out, with a log probability of -inf"""
    for at in (0, 5, 69, vocab // 2, vocab - 2, vocab - 1):
        c = make(rows, vocab, 128, dev)
        c["a"][:, 0] = 100
        c["b"][:, at] = 0
        c["b"][0, at] = -1
        c["b_scales"][at] = float("inf")
        c["tokens"][rows // 2] = at
        check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)
        # and whole tiles of them
        c["b"][:, 64:500] = 0
        c["b"][0, 64:500] = -1
        c["b_scales"][64:500] = float("inf")
        check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab", [600, 1003])
def test_negative_and_zero_scales(dev, rows, vocab):
    c = make(rows, vocab, 256, dev)
    c["a_scales"][::3] *= -1
    c["b_scales"][::5] *= -1
    if rows > 1:
        c["a_scales"][1] = 0
        c["a_scales"][rows - 1] = -0.0
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=vocab), c, vocab, 1)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", [1e6, 1e10, 1e20, 1e30])
def test_very_large_logits(dev, rows, size):
    """Whole tiles and a ragged one; both signs of the row's scale.  Of that size one token has all of the weight, or several of the same logit."""
    c = make(rows, 1003, 256, dev, size=size)
    if rows > 1:
        c["a_scales"][1] *= -1
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=1003), c, 1003, 1)
    c["b"][:, 8:1000] = c["b"][:, :8].repeat(1, 124)
    c["b_scales"][:1000] = c["b_scales"][0].clone()
    check(ops.scaled_mm_token_logprobs(**c, top=1, vocab=1003), c, 1003, 1)


@pytest.mark.parametrize("rows", [2, 70, 300])
def test_a_row_whose_logits_are_all_masked(dev, rows):
    c = make(rows, 500, 128, dev)
    c["a"][:, 0] = 100
    c["b"][:] = 0
    c["b"][0] = -1
    c["b_scales"][:500] = float("inf")
    got = ops.scaled_mm_token_logprobs(**c, top=1, vocab=500)
    assert all(torch.isnan(t).all() for t in got[:3]) and ((got.top_tokens >= 0) & (got.top_tokens < 500)).all()
    assert torch.isneginf(logits_of(c, 500)).all()
