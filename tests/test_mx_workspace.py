"""The workspace of a 4-bit product goes by m, n, k and a_type, as include/quamba_amd_mx.h says: whatever else the block holds (CPU)."""
import ctypes as C

import pytest

from quamba_amd import _lib


@pytest.mark.parametrize("a_type", ["QA_LM_F16", "QA_LM_BF16", "QA_LM_F32"])
@pytest.mark.parametrize("m,n,k", [(100, 100, 1024), (17, 50280, 2560), (1021, 50277, 1536)])
def test_sizes_and_the_rows_type_are_enough(a_type, m, n, k):
    l = _lib.lib()
    p = _lib.QaMxGemmParams()
    p.m, p.n, p.k, p.a_type = m, n, k, getattr(_lib, a_type)
    need = m * (k // 2 + 16 * -(-k // 512))                         # codes, and 16 scales for each group
    for out_type in (0, _lib.QA_LM_F16, _lib.QA_LM_BF16, _lib.QA_LM_F32, 77):
        p.out_type = out_type
        assert l.qa_mxfp4_mm_workspace_bytes(C.byref(p)) == need, out_type


def test_sizes_that_are_refused_need_none():
    l = _lib.lib()
    for fields in (dict(m=0), dict(n=0), dict(k=0), dict(m=-1), dict(k=1000), dict(k=(1 << 23) + 32), dict(m=(1 << 31) - 255), dict(a_type=4), dict(a_type=-1), dict(a_type=_lib.QA_LM_I8)):
        p = _lib.QaMxGemmParams()
        p.m, p.n, p.k, p.a_type, p.out_type = 100, 100, 1024, _lib.QA_LM_F16, _lib.QA_LM_F16
        for name, value in fields.items():
            setattr(p, name, value)
        assert l.qa_mxfp4_mm_workspace_bytes(C.byref(p)) == 0, fields
