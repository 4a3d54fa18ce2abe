"""The residual sum with its norms against the formula in 64 bits.

The kernel works in fp32.  Unit: 2^-24.  A sum of squares is a chain of at most 32 terms a lane, six lane exchanges and at most 15 more
waves, so 55 units, half of it in the reciprocal root; that root, the products of a norm, a gate (expf and a division) and the fused sum
add some 15.  v = r + s u is then within 45 units of |r| + |s u|, y within 45 of v's and as much for the norm over v, whose error is the
former's share of |v|: twice as much for operands of independent sign.  2^-16 (256 units) of (|r| + |s u|) |w| / rms(v) covers it; a rounding to a
narrower type adds half a step, an int8 code half of one."""
import numpy as np
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -16
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _wide(t):
    return t.detach().cpu().double().numpy()


def reference(x, weight, eps, residual=None, post_weight=None, gate=None, gate_act="none", residual_scale=1.0):
    """(y, v, |r| + |s u| as y sees it) in 64 bits"""
    u = _wide(x)
    if post_weight is not None:
        u = u / np.sqrt((u * u).mean(-1, keepdims=True) + eps) * _wide(post_weight)
    if gate is not None:
        g = _wide(gate)
        u = u * {"none": g, "sigmoid": 1 / (1 + np.exp(-g)), "silu": g / (1 + np.exp(-g))}[gate_act]
    u = u * (_wide(residual_scale) if torch.is_tensor(residual_scale) else residual_scale)
    r = 0.0 if residual is None else _wide(residual)
    v = r + u
    of_v = _wide(weight) / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return v * of_v, v, np.abs(r) + np.abs(u), np.abs(of_v)


def half_step(dtype, value):
    info = torch.finfo(dtype)
    return np.maximum(np.abs(value) * info.eps / 2, info.smallest_normal * info.eps / 2)


def check(got, want, x, out_scale=None):
    (y, v, scales), (y64, v64, size, of_v) = got, want
    if v is not None:
        assert np.all(np.abs(_wide(v) - v64) <= F32 * size + half_step(v.dtype, v64) * (1 + F32))
    off = F32 * size * of_v
    if y.dtype != torch.int8:
        assert y.dtype == x.dtype
        assert np.all(np.abs(_wide(y) - y64) <= off + half_step(y.dtype, y64) * (1 + F32))
        return
    if out_scale is None:
        most = np.abs(y64).max(-1)
        assert np.all(np.abs(_wide(scales) - np.maximum(most, 1e-5) / 127) <= (off.max(-1) + most * 2.0 ** -22) / 127)
        s = _wide(scales)[:, None]
    else:
        s = np.float64(np.float32(out_scale))
    exact = np.clip(y64 / s, -128, 127)
    assert np.all(np.abs(_wide(y) - exact) <= 0.5 + off / s + np.abs(exact) * 2.0 ** -22)


def make(rows, dim, dtype, dev, seed=0, residual="same", param="same", post=False, gate=None, scale=1.0):
    g = torch.Generator().manual_seed(1000 * rows + dim + seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    pt = dtype if param == "same" else torch.float32
    a = dict(x=r(rows, dim).to(dtype).to(dev), weight=(1 + 0.3 * r(dim)).to(pt).to(dev))
    if residual:
        a["residual"] = (2 * r(rows, dim)).to(dtype if residual == "same" else torch.float32).to(dev)
    if post:
        a["post_weight"] = (1 + 0.3 * r(dim)).to(pt).to(dev)
    if gate:
        a["gate"], a["gate_act"] = r(*((rows, dim) if gate[0] == "rows" else (dim,))).to(dtype).to(dev), gate[1]
    a["residual_scale"] = (0.5 + 0.1 * r(dim)).to(pt).to(dev) if scale == "channels" else scale
    return a


def call(a, **more):
    a = dict(a)
    return ops.add_rmsnorm(a.pop("x"), a.pop("weight"), 1e-5, **a, **more)


def want_of(a):
    a = dict(a)
    return reference(a.pop("x"), a.pop("weight"), 1e-5, **a)


# the narrowest row, rows of one lane and of one wave with a value more or less, waves that share a row, several pieces a lane, the widest
DIMS = [8, 9, 15, 64, 511, 512, 513, 768, 1000, 1531, 2560, 4099, 8192, 8200, 16391, 32761, 32768]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_sum_and_norm(dev, dim, dtype):
    a = make(5, dim, TYPES[dtype], dev)
    check(call(a), want_of(a), a["x"])


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 257, 2051])
@pytest.mark.parametrize("dim", [100, 512, 768, 2560])
def test_numbers_of_rows(dev, rows, dim):
    a = make(rows, dim, torch.float16, dev, residual="fp32")
    check(call(a, out_dtype=torch.int8), want_of(a), a["x"])


@pytest.mark.parametrize("dim", [77, 768, 2563, 8192, 20003])
@pytest.mark.parametrize("dtype,residual,param", [("fp16", "same", "fp32"), ("fp16", "fp32", "same"), ("bf16", "fp32", "fp32"), ("bf16", None, "same"),
                                                  ("fp32", "same", "same"), ("fp32", None, "same")])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
def test_a_block_with_everything(dev, dim, dtype, residual, param, act):
    """A norm behind the block, a gate of each kind, a scale per channel; each kind of output."""
    for kind in ("rows", "channels"):
        a = make(6, dim, TYPES[dtype], dev, residual=residual, param=param, post=True, gate=(kind, act), scale="channels")
        want = want_of(a)
        check(call(a), want, a["x"])
        check(call(a, out_dtype=torch.int8), want, a["x"])
        check(call(a, out_dtype=torch.int8, out_scale=0.031), want, a["x"], 0.031)


@pytest.mark.parametrize("post,gate,scale", [(True, None, 1.0), (False, ("rows", "silu"), 1.0), (False, None, 0.22), (False, None, "channels"), (True, None, -1.5)])
def test_each_part_alone(dev, post, gate, scale):
    a = make(9, 1100, torch.bfloat16, dev, residual="fp32", post=post, gate=gate, scale=scale)
    check(call(a), want_of(a), a["x"])


def test_rows_that_lie_apart(dev):
    """Rows cut out of wider ones, on any address; a gate that is one row for all, however it is given."""
    for shift in (0, 1, 3, 8):
        for dim in (768, 515):
            a = make(7, dim, torch.float16, dev, residual="fp32", post=True, gate=("rows", "silu"))
            for k in ("x", "residual", "gate"):
                t = torch.full((7, dim + 24), 7.0, dtype=a[k].dtype, device=dev)
                t[:, shift:shift + dim] = a[k]
                a[k] = t[:, shift:shift + dim]
            w = torch.ones(dim + 9, dtype=torch.float16, device=dev)
            w[shift:shift + dim] = a["weight"]
            a["weight"] = w[shift:shift + dim]
            out = torch.full((7, dim + 24), 5.0, device=dev)
            check(call(a, residual_out=out[:, shift:shift + dim]), want_of(a), a["x"])
            assert (out[:, :shift] == 5).all() and (out[:, shift + dim:] == 5).all()
    a = make(4, 256, torch.float16, dev, gate=("channels", "sigmoid"))
    want = call(a)
    for g in (a["gate"][None], a["gate"].expand(4, 256), a["gate"].repeat(4, 1)):
        got = call({**a, "gate": g})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dim", [8, 520, 1531, 2560, 9001, 32768])
@pytest.mark.parametrize("post", [False, True])
def test_the_stream_in_place(dev, dim, post):
    a = make(33, dim, torch.bfloat16, dev, residual="fp32", post=post, scale=0.7)
    want = call(a)
    stream = a["residual"].clone()
    y, v, _ = call({**a, "residual": stream}, residual_out=stream)
    assert v.data_ptr() == stream.data_ptr()
    assert torch.equal(y, want[0]) and torch.equal(stream, want[1])


def test_without_the_stream(dev):
    a = make(5, 640, torch.float16, dev, residual="fp32")
    want = call(a)
    y, v, s = call(a, prenorm=False)
    assert v is None and s is None and torch.equal(y, want[0])
    b = make(5, 640, torch.float16, dev, residual=None, scale=2.0)
    y, v, _ = call(b, residual_dtype=torch.float32)
    assert v.dtype == torch.float32 and torch.equal(v, 2 * b["x"].float())
    assert call(b)[1].dtype == torch.float16
    # the order of x's columns does not depend on what is asked for
    assert torch.equal(y, call(b, prenorm=False)[0])


def test_rows_of_zeros_and_of_nan(dev):
    """Zeros stay zeros (the scale of their codes is the least there is); a NaN or an infinity stays in its row."""
    a = make(6, 700, torch.float16, dev, residual="fp32")
    clean = call(a, out_dtype=torch.int8)
    a["x"][1] = 0
    a["residual"][1] = 0
    a["x"][3, 17] = float("nan")
    a["x"][4, 699] = float("inf")
    y, v, s = call(a, out_dtype=torch.int8)
    assert (y[1] == 0).all() and (v[1] == 0).all() and s[1].item() == np.float32(1e-5) / np.float32(127)
    assert torch.isnan(s[3]) and torch.isnan(s[4])
    for i in (0, 2, 5):
        assert torch.equal(y[i], clean[0][i]) and torch.equal(v[i], clean[1][i]) and s[i] == clean[2][i]
    y = call(a)[0]
    assert torch.isnan(y[3:5]).all() and (y[1] == 0).all() and not torch.isnan(y[[0, 2, 5]]).any()


def test_saturated_codes(dev):
    a = make(3, 256, torch.float16, dev)
    y, _, _ = call(a, out_dtype=torch.int8, out_scale=0.004)
    assert y.min() == -128 and y.max() == 127
    check((y, None, None), want_of(a), a["x"], 0.004)


def test_no_rows(dev):
    y, v, s = call(make(0, 640, torch.float16, dev, gate=("rows", "silu")), out_dtype=torch.int8)
    assert y.shape == (0, 640) and v.shape == (0, 640) and s.shape == (0,)


def test_on_another_stream_and_replayed(dev):
    a = make(64, 2560, torch.float16, dev, residual="fp32", post=True, gate=("rows", "silu"))
    want = call(a, out_dtype=torch.int8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(a, out_dtype=torch.int8)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(a, out_dtype=torch.int8)
    for i in range(3):
        a["x"].copy_(torch.randn(64, 2560, device=dev))
        graph.replay()
        now = call(a, out_dtype=torch.int8)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, now)), i


def test_refusals(dev):
    a = make(4, 64, torch.float16, dev, residual="fp32")
    x, w, r = a["x"], a["weight"], a["residual"]
    for bad in (dict(weight=w[:32]), dict(weight=w.bfloat16()), dict(residual=r[:3]), dict(residual=r.bfloat16()), dict(residual=r.t().contiguous().t()),
                dict(gate=torch.zeros(4, 32, dtype=torch.float16, device=dev)), dict(gate=torch.zeros(4, 64, device=dev)), dict(post_weight=w.float()),
                dict(residual_scale=w.float()), dict(out_scale=0.1), dict(out_dtype=torch.int8, out_scale=0.0), dict(residual=r.cpu()),
                dict(residual_dtype=torch.float16), dict(prenorm=False, residual_out=torch.empty_like(r)), dict(residual_out=torch.empty_like(x)),
                dict(gate=x.expand(2, 4, 64))):
        with pytest.raises(RuntimeError):
            ops.add_rmsnorm(x, **{"weight": w, "eps": 1e-5, "residual": r, **bad})
    for bad in (dict(gate_act="tanh"), dict(out_dtype=torch.float32), dict(out_dtype=torch.bfloat16)):
        with pytest.raises(NotImplementedError):
            ops.add_rmsnorm(x, w, 1e-5, residual=r, **bad)
    with pytest.raises(NotImplementedError):
        ops.add_rmsnorm(x[:, :7], w[:7], 1e-5)
    with pytest.raises(RuntimeError):
        ops.add_rmsnorm(x.cpu(), w, 1e-5)
    # a stream that is written over something else that is read
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.add_rmsnorm(x, w, 1e-5, residual_out=x)
    wide = torch.zeros(5, 64, device=dev)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.add_rmsnorm(x, w, 1e-5, residual=wide[:4], residual_out=wide[1:])
