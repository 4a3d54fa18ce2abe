"""The tensors that the operators around the mixers return and write: their memory, their versions, how they may lie."""
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [500, 5000])
def test_large_answers_do_not_keep_each_other(dev, rows):
    """What is kept, or saved, of many rows is what it shows"""
    logits, tokens = torch.randn(rows, 100, device=dev), torch.zeros(rows, dtype=torch.int64, device=dev)
    a, b = torch.zeros(rows, 64, dtype=torch.int8, device=dev), torch.zeros(96, 64, dtype=torch.int8, device=dev).t()
    one = torch.ones(1, device=dev)
    for got in (ops.token_logprobs(logits, tokens, top=20), ops.scaled_mm_token_logprobs(a, b, one, one, tokens, top=1)):
        for t in got:
            assert t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0
        assert len({t.untyped_storage().data_ptr() for t in got}) == 4


@pytest.mark.parametrize("lead,top", [((1,), 5), ((3,), 1), ((), 3), ((2, 3), 20), ((0,), 4), ((7,), 0)])
def test_small_answers_lie_on_whole_words(dev, lead, top):
    logits, tokens = torch.randn(*lead, 100, device=dev), torch.zeros(lead, dtype=torch.int64, device=dev)
    got = ops.token_logprobs(logits, tokens, top=top)
    assert [t.shape for t in got] == [lead, lead, (*lead, top), (*lead, top)]
    assert all(t.data_ptr() % 16 == 0 and t.is_contiguous() for t in got)
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in got if t.numel())
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))


def test_a_stream_that_is_written_has_another_version(dev):
    """so that autograd notices where it saved what was there before"""
    x, w = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    stream = torch.randn(4, 64, device=dev)
    before = stream._version
    ops.add_rmsnorm(x, w, 1e-5, residual=stream)
    assert stream._version == before
    ops.add_rmsnorm(x, w, 1e-5, residual=stream, residual_out=stream)
    assert stream._version > before
    leaf = torch.ones(4, 64, device=dev, requires_grad=True)
    kept = torch.randn(4, 64, device=dev)
    product = leaf * kept
    ops.add_rmsnorm(x, w, 1e-5, residual=kept, residual_out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    # a view has its base's version; a stream of inference mode has none, there and outside
    base = torch.zeros(4, 96, device=dev)
    before = base._version
    ops.add_rmsnorm(x, w, 1e-5, residual_out=base[:, 16:80])
    assert base._version > before
    with torch.inference_mode():
        held = torch.zeros(4, 64, device=dev)
        ops.add_rmsnorm(x, w, 1e-5, residual=held, residual_out=held)
    want = held.clone()
    ops.add_rmsnorm(x, w, 1e-5, residual=held, residual_out=held)
    assert torch.equal(held, want + x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_that_lie_between_rows(dev, dtype):
    """x, stream and what is written side by side in one piece of memory"""
    g = torch.Generator().manual_seed(1)
    memory = torch.randn(9, 3 * 72, generator=g).to(dtype).to(dev)
    x, r, out = memory[:, :64], memory[:, 72:136], memory[:, 152:216]
    w = torch.ones(64, dtype=dtype, device=dev)
    want = ops.add_rmsnorm(x.contiguous(), w, 1e-5, residual=r.contiguous())
    rest = memory[:, 64:72].clone(), memory[:, 136:152].clone()
    got = ops.add_rmsnorm(x, w, 1e-5, residual=r, residual_out=out)
    assert torch.equal(got[0], want[0]) and torch.equal(out, want[1])
    got = ops.add_rmsnorm(x, w, 1e-5, residual=r, residual_out=r)
    assert torch.equal(got[0], want[0]) and torch.equal(r, want[1])
    # every other row of one piece, and the rows between them
    pairs = memory[:8].clone()
    want = ops.add_rmsnorm(pairs[::2, :64].contiguous(), w, 1e-5)
    got = ops.add_rmsnorm(pairs[::2, :64], w, 1e-5, residual_out=pairs[1::2, :64])
    assert torch.equal(got[0], want[0]) and torch.equal(pairs[1::2, :64], want[1])
    assert torch.equal(memory[:, 64:72], rest[0]) and torch.equal(memory[:, 136:152], rest[1])
    # columns that are shared, a gate of one row among them, rows of another pitch: refused
    for bad in (dict(residual_out=memory[:, 60:124]), dict(residual_out=memory[:, 10:74]), dict(residual=r, residual_out=memory[:, 100:164]),
                dict(gate=memory[2, 152:216], residual_out=out),
                dict(residual_out=memory.view(-1)[64:64 + 9 * 70].view(9, 70)[:, :64])):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.add_rmsnorm(x, w, 1e-5, **bad)
