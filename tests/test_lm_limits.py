"""Sizes that the operators around the mixers refuse on the host, beyond what test_lm_abi covers (no GPU needed)."""
import ctypes as C

import pytest

from quamba_amd import _lib

AT = 1 << 20                                                       # an address that nothing reads


def _head(rows, vocab, k):
    p = _lib.QaMmTokenLogprobsParams()
    p.rows, p.vocab, p.k, p.lda, p.ldw = rows, vocab, k, k, k
    p.a_scale_numel = p.w_scale_numel = 1
    p.token_bytes = 8
    p.a = p.w = p.a_scale = p.w_scale = p.tokens = p.logprobs = p.entropy = p.workspace = AT
    p.workspace_bytes = 0                                          # (what is not refused for its sizes is for this)
    return p


@pytest.mark.parametrize("k,status", [(131056, -6), (131072, -2), (1 << 20, -2), (1 << 22, -2)])
def test_sums_that_32_bits_do_not_hold(k, status):
    """k products of codes are at most 2^14 k: below 2^31 up to k = 131056"""
    assert (131056 << 14) < (1 << 31) <= (131072 << 14)
    l, p = _lib.lib(), _head(4, 1000, k)
    assert (l.qa_mm_token_logprobs_workspace_bytes(C.byref(p)) > 0) == (status == -6)
    assert l.qa_mm_token_logprobs(C.byref(p), None) == status


def test_rows_whose_join_a_launch_does_not_count():
    """16 rows for each workgroup of 256: 2^32 threads for the last 16 of 2^28 rows, refused before the tiles are enqueued"""
    l, p = _lib.lib(), _head(1 << 28, 16, 16)
    p.workspace_bytes = (1 << 63) - 1
    assert l.qa_mm_token_logprobs(C.byref(p), None) == -2
    p.rows -= 15
    assert l.qa_mm_token_logprobs(C.byref(p), None) == -2
