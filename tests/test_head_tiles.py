"""Every tile of the head's log probabilities in its steady state: depths of many k tiles and of a rest, ragged rows and columns, checked against
64 bits.  Which tile a size takes is the library's rule, evaluated here from its table, so that a change of the table that
leaves a tile without a test shows."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from quamba_amd import _lib, ops
from test_finite_masks_gpu import check as check_logprobs
from test_mm_token_logprobs_gpu import make

SOURCE = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quamba_amd", "csrc", "gemm_logprobs.hip")).read()
TABLE = [tuple(np.float32(x.rstrip("f")) for x in t) for t in
         re.findall(r"\{(\d+), (\d+), ([\d.]+f), ([\d.]+f), ([\d.]+f)\}", re.search(r"kTiles\[\] = \{(.*?)\};", SOURCE, re.S).group(1))]
NARROW, MIDDLE, WIDE, SQUARE, WIDE_OF_128, LARGE, LARGEST = range(7)


def _up(a, b):
    return -(-a // b)


def plan(rows, vocab, k, cus):
    """(tile, columns it takes)"""
    units = _up(k, 128)

    def even(width):
        places = _up(vocab, cus * width) * cus
        return _up(vocab, 16 * places) * 16
    if rows <= 64:
        columns = max(even(256), 64)
        if columns > 128 and units <= 8:
            return MIDDLE, 128
        return (NARROW if columns <= 64 else MIDDLE if columns <= 128 else WIDE), columns
    cost = {i: fixed + np.float32(_up(_up(rows, int(bm)) * _up(vocab, int(bn)), cus)) * (each + unit * np.float32(units))
            for i, (bm, bn, fixed, each, unit) in enumerate(TABLE) if i != WIDE}
    best = min(cost, key=cost.get)
    return best, even(256) if best == WIDE_OF_128 and rows <= 128 else int(TABLE[best][1])


def test_the_rule_is_the_library_s():
    """by the columns of a tile, which the size of the workspace shows"""
    assert len(TABLE) == 7
    l, p = _lib.lib(), _lib.QaMmTokenLogprobsParams()
    p.token_bytes = 8
    cus = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 256
    for rows in (1, 33, 64, 65, 90, 128, 129, 256, 700, 1021, 5000, 16384):
        for vocab in (600, 4000, 16000, 50277, 50280, 256000):
            for k in (128, 768, 1040, 1536, 2560, 4096):
                p.rows, p.vocab, p.k = rows, vocab, k
                assert l.qa_mm_token_logprobs_workspace_bytes(C.byref(p)) == rows * (16 * _up(vocab, plan(rows, vocab, k, cus)[1]) + 4), (rows, vocab, k)


# tile, rows, vocabulary, K: whole k tiles (turned, for the first three) and a rest of them, more of them than stages
SIZES = [(NARROW, 64, 10007, 2560), (NARROW, 5, 9000, 1040), (MIDDLE, 40, 20011, 2560), (MIDDLE, 64, 20011, 1040),
         (WIDE, 1, 50280, 2560), (WIDE, 33, 50280, 2560), (WIDE, 64, 50280, 2560), (WIDE, 64, 50277, 1040),
         (SQUARE, 1000, 4000, 2560), (SQUARE, 1000, 4003, 1040),
         (WIDE_OF_128, 65, 50280, 1040), (WIDE_OF_128, 100, 50277, 2560), (WIDE_OF_128, 128, 50280, 2560),
         (LARGE, 256, 50280, 2560), (LARGE, 250, 50277, 2576), (LARGEST, 1021, 50277, 1536), (LARGEST, 1021, 50277, 1552)]


def test_every_tile_is_tested():
    assert {s[0] for s in SIZES} == set(range(7))
    assert all(plan(*size, 256)[0] == tile for tile, *size in SIZES), [(tile, size, plan(*size, 256)) for tile, *size in SIZES]


@pytest.mark.gpu
@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("tile,rows,vocab,k", SIZES)
def test_deep_tiles(dev, tile, rows, vocab, k, signs):
    """signs: row scales that are negative, and 0; rows at the tiles' edges are compared, and some between them"""
    if torch.cuda.get_device_properties(dev).multi_processor_count == 256:
        assert plan(rows, vocab, k, 256)[0] == tile
    c = make(rows, vocab, k, dev)
    if signs:
        c["a_scales"][::3] *= -1
        c["a_scales"][rows // 2] = 0
    g = torch.Generator().manual_seed(rows)
    at = sorted({r for r in (0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 255, 256, 511, 512, rows // 2, rows - 2, rows - 1, *torch.randint(0, rows, (12,), generator=g).tolist())
                 if 0 <= r < rows})
    c["tokens"][at[0]], c["tokens"][at[-1]] = vocab - 1, 0
    acc = (c["a"][at].double() @ c["b"][:, :vocab].double()).float()
    logits = (c["a_scales"][at][:, None] * (c["b_scales"][:vocab] * acc)).cpu()
    answers = []
    for top in (0, 1):
        got = ops.scaled_mm_token_logprobs(**c, top=top, vocab=vocab)
        check_logprobs(ops.TokenLogprobs(*(t[at] for t in got)), logits, c["tokens"][at], top)
        assert torch.isfinite(got.logprobs).all() and torch.isfinite(got.entropy).all()
        answers.append(got)
    assert torch.equal(answers[0].logprobs, answers[1].logprobs) and torch.equal(answers[0].entropy, answers[1].entropy)
