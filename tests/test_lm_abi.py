"""CPU-side checks of the C ABI of the operators around the mixers (include/quamba_amd_lm.h): symbols, version, layouts of the
parameter blocks, and what each entry point refuses before any GPU call."""
import ctypes as C
import hashlib
import os
import re
import subprocess

import pytest

from quamba_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "quamba_amd_lm.h")
TEXT = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
BLOCKS = re.findall(r"\}\s*(Qa[A-Za-z0-9]+Params)\s*;", TEXT)
# what the header's parameter blocks looked like at each version (comments and spacing aside)
BLOCKS_OF_VERSION = {1: "55a3ed496ad149c6"}


def test_symbols_and_version():
    names = sorted(set(re.findall(r"\b(qa_[a-z0-9_]+)\s*\(", TEXT)))
    assert sorted(_lib.LM_SYMBOLS) == names
    l = _lib.lib()
    assert all(getattr(l, n) is not None for n in names)
    assert l.qa_lm_abi_version() == _lib.LM_ABI_VERSION == int(re.search(r"#define QA_LM_ABI_VERSION (\d+)", TEXT).group(1))


def test_a_library_of_another_version_is_refused(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LM_ABI_VERSION", _lib.LM_ABI_VERSION + 1)
    with pytest.raises(RuntimeError, match="ABI versions"):
        _lib.lib()


def test_a_changed_block_has_another_version():
    blocks = re.findall(r"typedef struct (?:Qa\w+Params) \{.*?\} \w+;", TEXT, flags=re.S)
    assert len(blocks) == len(BLOCKS) == 3
    assert BLOCKS_OF_VERSION[_lib.LM_ABI_VERSION] == hashlib.sha256(re.sub(r"\s+", " ", " ".join(blocks)).encode()).hexdigest()[:16]


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name in BLOCKS:
        lines.append(f'printf("{name} . %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in getattr(_lib, name)._fields_]
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{HEADER}"\nint main(void){{{"".join(lines)}return 0;}}\n')
    subprocess.run(["gcc", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    want = {(a, b): int(c) for a, b, c in (line.split() for line in out.strip().splitlines())}
    for name in BLOCKS:
        cls = getattr(_lib, name)
        assert want[(name, ".")] == C.sizeof(cls) == sum(C.sizeof(t) for _, t in cls._fields_), name      # (no padding, no field left out)
        for f, _ in cls._fields_:
            assert want[(name, f)] == getattr(cls, f).offset, f"{name}.{f}"


def _codes(call, block, cases):
    """The status of the call with each set of fields changed"""
    for fields, status in cases:
        p = type(block).from_buffer_copy(block)
        for k, v in fields.items():
            setattr(p, k, v)
        assert call(C.byref(p), None) == status, (fields, status)


AT = 1 << 20                                                       # an address that nothing reads


def test_add_rmsnorm_refusals():
    l = _lib.lib()
    assert l.qa_add_rmsnorm(None, None) == -1
    p = _lib.QaAddNormParams()
    p.rows, p.dim = 4, 64
    p.x_type = p.param_type = p.residual_type = p.out_type = _lib.QA_LM_F16
    p.x_row_stride = p.residual_row_stride = p.residual_out_row_stride = p.gate_row_stride = p.out_row_stride = 64
    p.x = p.weight = p.out = p.residual = p.residual_out = p.gate = p.post_weight = p.scale_vector = p.scales = AT
    _codes(l.qa_add_rmsnorm, p, [
        (dict(rows=-1), -2), (dict(dim=0), -2), (dict(dim=7), -4), (dict(dim=32769), -4), (dict(x_type=0), -4), (dict(x_type=4), -4),
        (dict(param_type=2), -4), (dict(residual_type=2), -4), (dict(residual_type=0), -4), (dict(out_type=2), -4), (dict(out_type=3), -4),
        (dict(gate_act=3), -4), (dict(gate_act=-1), -4), (dict(out_type=0, out_scale=0.0), -4), (dict(out_type=0, out_scale=1e-39), -4),
        (dict(out_type=0, out_scale=float("inf")), -4), (dict(out_type=0, out_scale=float("nan")), -4), (dict(x=0), -1), (dict(weight=0), -1), (dict(out=0), -1),
        (dict(out_type=0, dynamic_scale=1, scales=0), -1), (dict(x=AT + 1), -3), (dict(weight=AT + 1), -3), (dict(post_weight=AT + 1), -3),
        (dict(scale_vector=AT + 1), -3), (dict(gate=AT + 1), -3), (dict(residual=AT + 1), -3), (dict(residual_out=AT + 1), -3), (dict(out=AT + 1), -3),
        (dict(residual_type=3, residual=AT + 2), -3), (dict(out_type=0, dynamic_scale=1, scales=AT + 2), -3), (dict(x_row_stride=63), -3),
        (dict(x_row_stride=-64), -3), (dict(residual_row_stride=0), -3), (dict(residual_out_row_stride=0), -3), (dict(out_row_stride=63), -3),
        (dict(gate_row_stride=63), -3), (dict(rows=0, x=0, weight=0, out=0, residual=0), 0)])


def test_token_logprobs_refusals():
    l = _lib.lib()
    assert l.qa_token_logprobs(None, None) == -1 and l.qa_token_logprobs_workspace_bytes(None) == 0
    p = _lib.QaTokenLogprobsParams()
    p.rows, p.vocab, p.logits_type, p.token_bytes, p.top, p.row_stride = 1, 50280, _lib.QA_LM_F16, 8, 5, 50280
    p.logits = p.tokens = p.logprobs = p.entropy = p.top_logprobs = p.top_tokens = p.workspace = AT
    p.workspace_bytes = need = l.qa_token_logprobs_workspace_bytes(C.byref(p))
    assert need > 0                                                # (one row is cut into segments)
    _codes(l.qa_token_logprobs, p, [
        (dict(rows=-1), -2), (dict(vocab=0), -2), (dict(vocab=(1 << 30) + 1), -2), (dict(top=65), -4), (dict(top=-1), -4), (dict(vocab=4), -2), (dict(logits_type=0), -4),
        (dict(logits_type=4), -4), (dict(token_bytes=2), -4), (dict(logits=0), -1), (dict(tokens=0), -1), (dict(logprobs=0), -1), (dict(entropy=0), -1),
        (dict(top_logprobs=0), -1), (dict(top_tokens=0), -1), (dict(logits=AT + 1), -3), (dict(tokens=AT + 4), -3), (dict(rows=2, row_stride=50279), -3),
        (dict(workspace=0), -1), (dict(workspace=AT + 8), -6), (dict(workspace_bytes=need - 1), -6), (dict(rows=0, logits=0, tokens=0, workspace=0), 0)])
    p.rows = 0
    assert l.qa_token_logprobs_workspace_bytes(C.byref(p)) == 0
    p.rows, p.top = 1, 65
    assert l.qa_token_logprobs_workspace_bytes(C.byref(p)) == 0
    p.rows, p.top = 1 << 20, 5                                     # whole rows
    assert l.qa_token_logprobs_workspace_bytes(C.byref(p)) == 0


def test_mm_token_logprobs_refusals():
    l = _lib.lib()
    assert l.qa_mm_token_logprobs(None, None) == -1 and l.qa_mm_token_logprobs_workspace_bytes(None) == 0
    p = _lib.QaMmTokenLogprobsParams()
    p.rows, p.vocab, p.k, p.a_scale_numel, p.w_scale_numel, p.token_bytes, p.top, p.lda, p.ldw = 4, 1000, 256, 4, 1008, 8, 1, 256, 256
    p.a = p.w = p.a_scale = p.w_scale = p.tokens = p.logprobs = p.entropy = p.top_logprobs = p.top_tokens = p.workspace = AT
    p.workspace_bytes = need = l.qa_mm_token_logprobs_workspace_bytes(C.byref(p))
    assert need > 0
    _codes(l.qa_mm_token_logprobs, p, [
        (dict(rows=-1), -2), (dict(vocab=0), -2), (dict(k=0), -2), (dict(top=2), -4), (dict(top=-1), -4), (dict(token_bytes=1), -4), (dict(a=0), -1),
        (dict(w=0), -1), (dict(a_scale=0), -1), (dict(w_scale=0), -1), (dict(tokens=0), -1), (dict(logprobs=0), -1), (dict(entropy=0), -1),
        (dict(top_logprobs=0), -1), (dict(top_tokens=0), -1), (dict(workspace=0), -1), (dict(a_scale_numel=3), -2), (dict(w_scale_numel=999), -2),
        (dict(k=250, lda=256), -3), (dict(lda=264), -3), (dict(ldw=264), -3), (dict(lda=240), -3), (dict(ldw=240), -3), (dict(a=AT + 8), -3), (dict(w=AT + 8), -3),
        (dict(a_scale=AT + 2), -3), (dict(w_scale=AT + 2), -3), (dict(tokens=AT + 4), -3), (dict(vocab=(1 << 30) + 1), -2), (dict(lda=(1 << 22) + 16), -2),
        (dict(ldw=(1 << 22) + 16), -2), (dict(workspace=AT + 8), -6), (dict(workspace_bytes=need - 1), -6),
        (dict(rows=0, a=0, w=0, tokens=0, workspace=0), 0)])
    for bad in (dict(rows=0), dict(vocab=0), dict(k=0), dict(top=2)):
        q = _lib.QaMmTokenLogprobsParams.from_buffer_copy(p)
        for k, v in bad.items():
            setattr(q, k, v)
        assert l.qa_mm_token_logprobs_workspace_bytes(C.byref(q)) == 0


def test_launches_of_too_many_threads_are_refused():
    """Work that a launch cannot count: refused on the host, before anything is enqueued"""
    l, most = _lib.lib(), (1 << 31) - 1
    p = _lib.QaAddNormParams()
    p.x_type = p.param_type = p.residual_type = p.out_type = _lib.QA_LM_F16
    p.x = p.weight = p.out = AT
    for dim, rows in ((8, 1 << 26), (512, most), (2560, 1 << 25), (32768, 1 << 22)):
        p.rows, p.dim, p.x_row_stride, p.out_row_stride = rows, dim, dim, dim
        assert l.qa_add_rmsnorm(C.byref(p), None) == -2, (dim, rows)
    t = _lib.QaTokenLogprobsParams()
    t.logits_type, t.token_bytes, t.top = _lib.QA_LM_F16, 8, 1
    t.logits = t.tokens = t.logprobs = t.entropy = t.top_logprobs = t.top_tokens = AT
    for vocab, rows in ((8, 1 << 26), (8, most), (50280, most)):
        t.rows, t.vocab, t.row_stride = rows, vocab, vocab
        assert l.qa_token_logprobs_workspace_bytes(C.byref(t)) == 0 and l.qa_token_logprobs(C.byref(t), None) == -2, (vocab, rows)
    h = _lib.QaMmTokenLogprobsParams()
    h.k = h.lda = h.ldw = 16
    h.a_scale_numel = h.w_scale_numel = 1
    h.token_bytes = 8
    h.a = h.w = h.a_scale = h.w_scale = h.tokens = h.logprobs = h.entropy = h.workspace = AT
    for vocab, rows in ((16, (1 << 28) + 1), (16, most), (1 << 30, 1 << 20)):
        h.rows, h.vocab, h.workspace_bytes = rows, vocab, (1 << 63) - 1
        assert l.qa_mm_token_logprobs(C.byref(h), None) == -2, (vocab, rows)
