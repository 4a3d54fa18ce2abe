"""CPU-side checks of the C ABI of the microscaled 4-bit operators and of beam search (include/quamba_amd_mx.h, include/quamba_amd_beam.h): symbols,
versions, layouts of the parameter blocks, and what each entry point refuses before any GPU call."""
import ctypes as C
import hashlib
import os
import re
import subprocess

import pytest
import torch

from quamba_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = {n: os.path.join(ROOT, "include", f"quamba_amd_{n}.h") for n in ("mx", "beam")}
TEXTS = {n: re.sub(r"/\*.*?\*/", "", open(h).read(), flags=re.S) for n, h in HEADERS.items()}
BLOCKS = {n: re.findall(r"\}\s*(Qa[A-Za-z0-9]+)\s*;", t) for n, t in TEXTS.items()}
SYMBOLS = {"mx": _lib.MX_SYMBOLS, "beam": _lib.BEAM_SYMBOLS}
VERSIONS = {"mx": _lib.MX_ABI_VERSION, "beam": _lib.BEAM_ABI_VERSION}
# what the headers' parameter blocks looked like at each version (comments and spacing aside)
BLOCKS_OF_VERSION = {"mx": {1: "81dc0ea47043f483"}, "beam": {1: "1f5b63dbdea6b272"}}
AT = 1 << 20                                                       # an address that nothing reads


@pytest.mark.parametrize("n", sorted(HEADERS))
def test_symbols_and_version(n):
    names = sorted(set(re.findall(r"\b(qa_[a-z0-9_]+)\s*\(", TEXTS[n])))
    assert sorted(SYMBOLS[n]) == names
    l = _lib.lib()
    assert all(getattr(l, name) is not None for name in names)
    assert getattr(l, f"qa_{n}_abi_version")() == VERSIONS[n] == int(re.search(rf"#define QA_{n.upper()}_ABI_VERSION (\d+)", TEXTS[n]).group(1))


@pytest.mark.parametrize("version", ["MX_ABI_VERSION", "BEAM_ABI_VERSION"])
def test_a_library_of_another_version_is_refused(monkeypatch, version):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, version, getattr(_lib, version) + 1)
    with pytest.raises(RuntimeError, match="ABI versions"):
        _lib.lib()


@pytest.mark.parametrize("n", sorted(HEADERS))
def test_a_changed_block_has_another_version(n):
    blocks = re.findall(r"typedef struct (?:Qa\w+) \{.*?\} \w+;", TEXTS[n], flags=re.S)
    assert len(blocks) == len(BLOCKS[n]) == 3
    assert BLOCKS_OF_VERSION[n][VERSIONS[n]] == hashlib.sha256(re.sub(r"\s+", " ", " ".join(blocks)).encode()).hexdigest()[:16]


@pytest.mark.parametrize("n", sorted(HEADERS))
def test_struct_layouts_match_the_header(n, tmp_path):
    lines = []
    for name in BLOCKS[n]:
        lines.append(f'printf("{name} . %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in getattr(_lib, name)._fields_]
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{HEADERS[n]}"\nint main(void){{{"".join(lines)}return 0;}}\n')
    subprocess.run(["gcc", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    want = {(a, b): int(c) for a, b, c in (line.split() for line in out.strip().splitlines())}
    for name in BLOCKS[n]:
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


@pytest.mark.parametrize("name,block,numbers,stride,kind", [
    ("qa_mxfp4_quant", _lib.QaMxQuantParams, "x", "x_row_stride", "x_type"), ("qa_mxfp4_dequant", _lib.QaMxDequantParams, "out", "out_row_stride", "out_type")])
def test_quant_refusals(name, block, numbers, stride, kind):
    call = getattr(_lib.lib(), name)
    assert call(None, None) == -1
    p = block()
    p.rows, p.k, p.code_row_stride, p.scale_group_stride = 4, 1024, 512, 64
    setattr(p, kind, _lib.QA_LM_F16)
    setattr(p, stride, 1024)
    setattr(p, numbers, AT)
    p.codes = p.scales = AT
    _codes(call, p, [
        (dict(rows=-1), -2), (dict(k=-32), -2), (dict(k=1000), -2), (dict(k=16), -2), ({kind: 0}, -4), ({kind: 4}, -4), ({numbers: 0}, -1), (dict(codes=0), -1),
        (dict(scales=0), -1), ({numbers: AT + 1}, -3), ({numbers: AT + 2, kind: 3}, -3), ({stride: 1023}, -3), ({stride: -1024}, -3), (dict(codes=AT + 8), -3),
        (dict(scales=AT + 4), -3), (dict(code_row_stride=520), -3), (dict(code_row_stride=496), -3), (dict(scale_group_stride=72), -3), (dict(scale_group_stride=48), -3),
        (dict(rows=(1 << 31) - 1, scale_group_stride=1 << 40), -2), ({"rows": 0, "codes": 0, "scales": 0, numbers: 0}, 0), ({"k": 0, "codes": 0, "scales": 0, numbers: 0}, 0)])


def test_mm_refusals():
    l = _lib.lib()
    assert l.qa_mxfp4_mm(None, None) == -1 and l.qa_mxfp4_mm_workspace_bytes(None) == 0
    p = _lib.QaMxGemmParams()
    p.m, p.n, p.k, p.a_type, p.out_type = 4, 100, 1024, _lib.QA_LM_I8, _lib.QA_LM_F16
    p.lda = p.ldw = 512
    p.ldd, p.a_scale_group_stride, p.w_scale_group_stride = 100, 64, 1600
    p.a = p.a_scales = p.w = p.w_scales = p.d = AT
    assert l.qa_mxfp4_mm_workspace_bytes(C.byref(p)) == 0
    _codes(l.qa_mxfp4_mm, p, [
        (dict(m=-1), -2), (dict(n=-1), -2), (dict(k=-32), -2), (dict(k=1000), -2), (dict(a_type=4), -4), (dict(a_type=-1), -4), (dict(out_type=0), -4), (dict(out_type=4), -4),
        (dict(a=0), -1), (dict(a_scales=0), -1), (dict(w=0), -1), (dict(w_scales=0), -1), (dict(d=0), -1), (dict(a=AT + 8), -3), (dict(a_scales=AT + 8), -3), (dict(w=AT + 8), -3),
        (dict(w_scales=AT + 8), -3), (dict(d=AT + 1), -3), (dict(out_type=3, d=AT + 2), -3), (dict(lda=520), -3), (dict(lda=496), -3), (dict(ldw=520), -3), (dict(ldw=496), -3),
        (dict(ldd=99), -3), (dict(a_scale_group_stride=48), -3), (dict(a_scale_group_stride=72), -3), (dict(w_scale_group_stride=1584), -3), (dict(w_scale_group_stride=1608), -3),
        (dict(lda=(1 << 24) + 16), -2), (dict(ldw=(1 << 24) + 16), -2), (dict(k=(1 << 25) + 32, lda=1 << 25, ldw=1 << 25), -2),
        (dict(lda=(1 << 22) + 16), -2), (dict(ldw=(1 << 22) + 16), -2), (dict(m=(1 << 31) - 255), -2), (dict(n=(1 << 31) - 255, ldd=1 << 31), -2),
        (dict(k=0, ldd=104), -3), (dict(m=0, a=0, w=0, d=0), 0), (dict(n=0, a=0, w=0, d=0), 0)])
    # rows of numbers: codes of their own where the rows are many
    p.m, p.a_type, p.lda, p.a_scales = 100, _lib.QA_LM_BF16, 1024, None
    p.workspace_bytes = need = l.qa_mxfp4_mm_workspace_bytes(C.byref(p))
    assert need == 100 * (512 + 2 * 16)
    p.workspace = AT
    _codes(l.qa_mxfp4_mm, p, [(dict(a=AT + 1), -3), (dict(lda=1023), -3), (dict(workspace=0), -1), (dict(workspace=AT + 8), -6), (dict(workspace_bytes=need - 1), -6)])
    p.m = 1
    assert l.qa_mxfp4_mm_workspace_bytes(C.byref(p)) == 0
    p.m, p.k = 100, 1000
    assert l.qa_mxfp4_mm_workspace_bytes(C.byref(p)) == 0


def test_beam_refusals():
    l = _lib.lib()
    assert l.qa_beam_search_step(None, None) == -1 and l.qa_beam_search_workspace_bytes(None) == 0
    p = _lib.QaBeamSearchParams()
    p.batch, p.beams, p.vocab, p.logits_type, p.count = 2, 4, 50280, _lib.QA_LM_F16, 8
    p.logits_beam_stride, p.logits_batch_stride = 50280, 4 * 50280
    p.logits = p.scores = p.out_scores = p.tokens = p.parents = p.workspace = AT
    p.workspace_bytes = need = l.qa_beam_search_workspace_bytes(C.byref(p))
    assert need > 0
    _codes(l.qa_beam_search_step, p, [
        (dict(batch=-1), -2), (dict(beams=0), -2), (dict(beams=65), -4), (dict(vocab=0), -2), (dict(vocab=(1 << 20) + 1), -2), (dict(count=0), -4), (dict(count=65), -4),
        (dict(vocab=1, count=5), -2), (dict(logits_type=0), -4), (dict(logits_type=4), -4), (dict(logits=0), -1), (dict(scores=0), -1), (dict(out_scores=0), -1),
        (dict(tokens=0), -1), (dict(parents=0), -1), (dict(logits=AT + 1), -3), (dict(logits_type=3, logits=AT + 2), -3), (dict(scores=AT + 2), -3),
        (dict(logits_beam_stride=-1), -3), (dict(logits_batch_stride=-1), -3), (dict(workspace=0), -1), (dict(workspace=AT + 8), -6), (dict(workspace_bytes=need - 1), -6),
        (dict(batch=1 << 30), -2), (dict(batch=1 << 24, workspace_bytes=(1 << 63) - 1), -2), (dict(batch=0, logits=0, scores=0, workspace=0), 0)])
    for bad in (dict(batch=0), dict(beams=0), dict(beams=65), dict(count=65), dict(vocab=0)):
        q = _lib.QaBeamSearchParams.from_buffer_copy(p)
        for k, v in bad.items():
            setattr(q, k, v)
        assert l.qa_beam_search_workspace_bytes(C.byref(q)) == 0


def test_reorder_refusals():
    l = _lib.lib()
    assert l.qa_reorder_states(None, None) == -1
    rows = (_lib.QaStateRows * 2)()
    for r in rows:
        r.data, r.row_bytes, r.row_stride = AT, 256, 256
    p = _lib.QaReorderParams()
    p.batch, p.beams, p.tensors, p.index_bytes, p.states, p.parents = 2, 4, 2, 8, rows, AT
    _codes(l.qa_reorder_states, p, [
        (dict(batch=-1), -2), (dict(beams=0), -2), (dict(beams=65), -4), (dict(tensors=-1), -2), (dict(index_bytes=2), -4), (dict(parents=0), -1), (dict(parents=AT + 4), -3),
        (dict(batch=65536), -2), (dict(batch=0, parents=0), 0), (dict(tensors=0, parents=0), 0), (dict(beams=1), 0)])
    p.states = None
    assert l.qa_reorder_states(C.byref(p), None) == -1
    p.states = rows
    for fields, status in ((dict(data=0), -1), (dict(row_bytes=-1), -2), (dict(row_stride=255), -3), (dict(row_stride=-256), -3), (dict(row_bytes=1 << 40, row_stride=1 << 40), -2),
                           (dict(row_bytes=(1 << 35) + 1, row_stride=1 << 36), -2)):
        for k, v in fields.items():
            setattr(rows[1], k, v)
        assert l.qa_reorder_states(C.byref(p), None) == status, (fields, status)
        rows[1].data, rows[1].row_bytes, rows[1].row_stride = AT, 256, 256


def test_the_python_layer_refuses_cpu_tensors():
    x, codes, scales = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 2, 16, dtype=torch.uint8)
    for call in (lambda: ops.mxfp4_quant(x), lambda: ops.mxfp4_dequant(codes, scales), lambda: ops.mxfp4_mm(codes, scales, codes, scales),
                 lambda: ops.mxfp4_linear(x, codes, scales), lambda: ops.beam_search_step(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2),
                 lambda: ops.reorder_states([x], torch.zeros(1, 2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        ops.mxfp4_quant(None)


@pytest.mark.parametrize("rows,blocks", [(1, 1), (3, 16), (2, 17), (5, 80), (4, 33)])
def test_orders_of_scales(rows, blocks):
    """block 4 j + q of a group at place 4 q + j, zeros behind the last one, and back"""
    natural = torch.randint(0, 255, (rows, blocks), dtype=torch.uint8)
    laid = ops.mxfp4_scales(natural)
    assert laid.shape == (-(-blocks // 16), rows, 16) and laid.is_contiguous()
    for g in range(laid.shape[0]):
        for j in range(4):
            for q in range(4):
                b = 16 * g + 4 * j + q
                want = natural[:, b] if b < blocks else torch.zeros(rows, dtype=torch.uint8)
                assert torch.equal(laid[g, :, 4 * q + j], want)
    assert torch.equal(ops.mxfp4_scales_of(laid, blocks), natural)
    for bad in (lambda: ops.mxfp4_scales(natural[0]), lambda: ops.mxfp4_scales(natural.int()), lambda: ops.mxfp4_scales_of(laid, 16 * laid.shape[0] + 1),
                lambda: ops.mxfp4_scales_of(natural, 1)):
        with pytest.raises(RuntimeError):
            bad()
