"""Beam selection where scores meet a border: one token that has all of its beam's weight, beams whose distributions are the same one.

A row of which one token has all the weight gives that token the beam's own score, whatever its logit: l - l - log 1.  So equal scores stay equal, and the lower beam
comes first.  Rows whose logits differ by one number that is exact in their type have the same differences from their largest logit, hence the same scores, bit for bit."""
import numpy as np
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
VOCABS = [3, 40, 2048, 2051, 50280, 200001]                        # less than a load, one chunk, one more value, several segments


def drawn(g, count, vocab):
    return torch.randperm(vocab, generator=g)[:count]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("mask", ["-inf", "lowest", "below"])
@pytest.mark.parametrize("far", [0.0, 3000.0, 5e6])
def test_one_token_has_all_the_weight(dev, dtype, vocab, mask, far):
    """that token has the score of its beam, and of beams with equal scores the lower comes first; other tokens' are masked or a hundred below"""
    if dtype == "fp16" and far > 3000:
        pytest.skip("beyond the type")
    g = torch.Generator().manual_seed(vocab + int(far))
    batch, beams = 3, 4
    for sign in (1.0, -1.0):
        allowed = torch.stack([drawn(g, 1, vocab) for _ in range(batch * beams)]).view(batch, beams, 1)
        own = (sign * far + 3 * torch.randn(batch, beams, 1, generator=g)).to(TYPES[dtype])
        if mask == "below":
            step = 100.0 if far < 1e6 else 2.0 ** 17                # (a step of the type at least)
            logits = (own.float() - step - step * torch.rand(batch, beams, vocab, generator=g)).to(TYPES[dtype])
        else:
            logits = torch.full((batch, beams, vocab), float("-inf") if mask == "-inf" else torch.finfo(TYPES[dtype]).min, dtype=TYPES[dtype])
        logits = logits.scatter_(2, allowed, own).to(dev)
        for scores in (torch.zeros(batch, beams), torch.full((batch, beams), -7.25), torch.tensor([-1.0, -3.0, -1.0, -3.0]).expand(batch, beams)):
            got = ops.beam_search_step(logits, scores.to(dev), beams)
            order = torch.sort(scores, dim=1, descending=True, stable=True).indices
            assert got.parents.tolist() == order.tolist()
            assert got.tokens.tolist() == allowed[..., 0].gather(1, order).tolist()
            assert torch.equal(got.scores.cpu(), scores.gather(1, order))
            # more places than that: the same ones first
            more = ops.beam_search_step(logits, scores.to(dev), 2 * beams)
            assert all(torch.equal(a[:, :beams], b) for a, b in zip(more, got))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("allowed", [2, 3, 7])
def test_equal_logits_share_the_weight(dev, dtype, vocab, allowed):
    """of `allowed` tokens with one logit, another in each beam and elsewhere: scores of log(1 / allowed), beam by beam, token by token"""
    if allowed > vocab:
        pytest.skip("more than there are")
    g = torch.Generator().manual_seed(vocab + allowed)
    logits = torch.full((1, 5, vocab), float("-inf"), dtype=TYPES[dtype])
    tokens = []
    for i in range(5):
        at = drawn(g, allowed, vocab).sort().values
        logits[0, i, at] = (4 * torch.randn(1, generator=g)).to(TYPES[dtype])
        tokens += at.tolist()
    got = ops.beam_search_step(logits.to(dev), torch.zeros(1, 5, device=dev), 5 * allowed)
    assert got.parents[0].tolist() == [i for i in range(5) for _ in range(allowed)] and got.tokens[0].tolist() == tokens
    assert torch.equal(got.scores.cpu(), torch.full((1, 5 * allowed), -np.log(allowed)))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [3, 40, 2051, 50280])
@pytest.mark.parametrize("masked", [False, True])
def test_rows_that_differ_by_a_number(dev, dtype, vocab, masked):
    """the same distribution in every beam: each token of all beams, the lower beam first, then the next token"""
    g = torch.Generator().manual_seed(vocab)
    row = torch.randint(-15, 16, (vocab,), generator=g) / 8.0      # (with what is added a multiple of 1 / 8 below 16: seven bits and a sign)
    row[torch.randperm(vocab, generator=g)[0]] = 2.25
    if masked:
        row[torch.randperm(vocab, generator=g)[:vocab // 3]] = float("-inf")
    added = torch.tensor([0.0, 1.25, -9.5, 7.75, -3.125, 12.0])
    logits = (row + added[:, None])[None].to(TYPES[dtype])
    assert torch.equal(logits.float(), (row + added[:, None])[None])
    count = min(int(row.isfinite().sum()), 6) * 6
    got = ops.beam_search_step(logits.to(dev), torch.full((1, 6), -2.5, device=dev), count)
    # (equal logits in one beam come before the next beam's)
    values, order = torch.sort(row, descending=True, stable=True)
    want = []
    for v in torch.unique(values[values.isfinite()]).flip(0):
        want += [(i, t) for i in range(6) for t in order[values == v].tolist()]
    assert list(zip(got.parents[0].tolist(), got.tokens[0].tolist())) == want[:count]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [3, 2051, 50280])
def test_no_score_above_its_beams(dev, dtype, vocab):
    """most of the weight on one token, more or less of it"""
    g = torch.Generator().manual_seed(vocab)
    for gap in (1.0, 5.0, 20.0, 30.0, 36.0, 40.0):
        logits = torch.randn(8, 4, vocab, generator=g) - gap
        logits.scatter_(2, torch.randint(0, vocab, (8, 4, 1), generator=g), torch.randn(8, 4, 1, generator=g))
        got = ops.beam_search_step(logits.to(TYPES[dtype]).to(dev), torch.zeros(8, 4, device=dev), 8)
        assert (got.scores <= 0).all()


def test_masks_of_the_lowest_value_beside_minus_infinity(dev):
    """two tokens at the type's least finite value have all there is, also beside -inf"""
    for dtype in TYPES.values():
        for vocab in (40, 50280):
            logits = torch.full((1, 2, vocab), float("-inf"), dtype=dtype, device=dev)
            logits[0, :, 7] = logits[0, :, vocab - 2] = torch.finfo(dtype).min
            got = ops.beam_search_step(logits, torch.zeros(1, 2, device=dev), 6)
            assert got.parents[0].tolist() == [0, 0, 1, 1, -1, -1] and got.tokens[0].tolist() == [7, vocab - 2] * 2 + [-1, -1]
            assert torch.equal(got.scores[0, :4].cpu(), torch.full((4,), -np.log(2.0), dtype=torch.float32))
            # and neighbouring finite values far from 0: the larger alone
            logits[0, :, 7] = torch.nextafter(torch.tensor(torch.finfo(dtype).min, dtype=dtype), torch.tensor(0.0, dtype=dtype)) if dtype != torch.float16 else -60000.0
            got = ops.beam_search_step(logits, torch.zeros(1, 2, device=dev), 2)
            assert got.tokens[0].tolist() == [7, 7] and got.scores[0].tolist() == [0.0, 0.0]
