"""Beam selection where a score is next to 0, so that what is written shows the error of the sums.

A term is off by less than 9e-15 of itself (the first missing term of its polynomial, r^4 / 24 with r up to ln 2 / 1024) and 2.5e-15 (18 roundings
of 1.1e-16 of its power of two and 5 of the polynomial and the product), the term that the sum is divided by as much, and a dozen additions, divisions and the sums of logits up to
16 and of a score up to 16 take 16 roundings of at most 2^-53 * 16: 5.2e-14 together, and half a step of fp32."""
import numpy as np
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [3, 2051, 50280])
@pytest.mark.parametrize("allowed", [2, 3])
def test_scores_next_to_zero(dev, vocab, allowed):
    """a beam's own score that nearly takes its best token's log probability away: what is left shows the sum's error"""
    g = torch.Generator().manual_seed(10 * vocab + allowed)
    batch, beams = 40, 4
    logits = torch.full((batch, beams, vocab), float("-inf"))
    for b in range(batch):
        for i in range(beams):
            logits[b, i, torch.randperm(vocab, generator=g)[:allowed]] = 3 * torch.rand(allowed, generator=g) - 8
    l = logits.numpy().astype(np.longdouble)
    most = l.max(-1, keepdims=True)
    best = -np.log(np.exp(l - most).sum(-1))                       # log probability of the best token, in 64 bits of mantissa
    own = (-best).astype(np.float32)
    got = ops.beam_search_step(logits.to(dev), torch.from_numpy(own).to(dev), beams * allowed)
    for b in range(batch):
        for score, token, parent in zip(*(t[b].tolist() for t in got)):
            if token != int(l[b, parent].argmax()):
                continue
            want = own[b, parent].astype(np.longdouble) + best[b, parent]
            assert abs(score - want) <= 5.2e-14 + abs(want) * 2.0 ** -24, (b, parent, score, float(want))
