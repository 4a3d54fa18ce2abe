"""Products of microscaled 4-bit operands against 64 bits.

With scales from 1 to 4 all products are multiples of 1/4 below 36 * 16, so up to K = 4096 every sum, in whatever order, is a multiple of 1/4 below 2^22: exact in
fp32, and the product has to be that number, rounded once to the output's type.

Otherwise: an instruction adds 128 products to the sum so far.  It keeps 26 bits at least below the largest of them (what it drops is less than 2^-26 of that
each, 129 numbers) and rounds to fp32 (2^-24), which is less than 2^-18 of S = sum |a| |w| an instruction; the sums of parts add a rounding each."""
import numpy as np
import pytest
import torch

from launched import expect, kernels
from mxfp4_reference import operand
from quamba_amd import MXFP4Linear, ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = [(1, 1, 32), (1, 16, 64), (1, 10, 768), (1, 2560, 2560), (2, 100, 96), (3, 257, 512), (5, 48, 544), (15, 33, 1056), (16, 64, 160), (17, 130, 480), (31, 1000, 1536),
         (32, 96, 2048), (33, 31, 992), (48, 1537, 768), (63, 65, 1024), (64, 500, 2560), (64, 4100, 256), (65, 127, 352), (96, 200, 4096), (127, 129, 1248), (128, 128, 1024),
         (129, 384, 608), (200, 777, 2592), (255, 257, 512), (256, 256, 1536), (257, 1000, 736), (384, 513, 2080), (500, 2560, 640), (511, 640, 3104), (1000, 1111, 288),
         (1021, 50, 1536), (2049, 300, 416), (40, 20000, 96), (3000, 17, 768), (300, 5000, 32), (700, 3001, 1024), (4300, 4201, 1024), (4300, 4201, 160), (4300, 5501, 1536), (600, 50001, 512), (12000, 1501, 1536)]


def exact_case(g, m, n, k, dev):
    a, a_scales, a_values = operand(g, m, k, 0, 2, dev)
    w, w_scales, w_values = operand(g, n, k, 0, 2, dev)
    return a, a_scales, w, w_scales, torch.from_numpy(a_values @ w_values.T)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_sums(dev, m, n, k):
    a, a_scales, w, w_scales, want = exact_case(np.random.default_rng(m * n + k), m, n, k, dev)
    for name, dtype in TYPES.items():
        got = ops.mxfp4_mm(a, a_scales, w, w_scales, out_dtype=dtype)
        assert got.shape == (m, n) and got.dtype == dtype
        assert torch.equal(got.cpu(), want.to(torch.float32).to(dtype)), name


@pytest.mark.parametrize("m,n,k", [(1, 500, 4096), (4, 130, 10240), (16, 1000, 2560), (33, 200, 5120), (64, 700, 8192), (130, 300, 2560), (300, 520, 5120), (600, 700, 1536)])
@pytest.mark.parametrize("spread", [0, 12])
def test_sums_that_round(dev, m, n, k, spread):
    """blocks of any sizes beside each other"""
    g = np.random.default_rng(m + n + k + spread)
    a, a_scales, a_values = operand(g, m, k, -spread, spread, dev)
    w, w_scales, w_values = operand(g, n, k, -spread, spread, dev)
    want, size = a_values @ w_values.T, np.abs(a_values) @ np.abs(w_values).T
    instructions = (k + 127) // 128
    for dtype in TYPES.values():
        half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
        got = ops.mxfp4_mm(a, a_scales, w, w_scales, out_dtype=dtype).cpu().double().numpy()
        most = torch.finfo(dtype).max
        least = torch.finfo(dtype).smallest_normal * half * 2
        fine = np.abs(want) + size * 2.0 ** -12 < most
        bound = size * (2.0 ** -18 * instructions + 2.0 ** -24 * 16) * (1 + half) + np.abs(want) * half + least
        assert np.all(np.abs(got - want)[fine] <= bound[fine])
        # (and far inside on average: what is dropped is of either sign, rounded sums are off by a third of a half step; where the type holds any)
        assert not fine.any() or np.abs(got - want)[fine].mean() <= (size * 2.0 ** -24 * instructions + np.abs(want) * half)[fine].mean()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 500, 768), (3, 33, 32), (7, 40, 544), (16, 100, 2560), (17, 64, 1536), (64, 300, 96), (200, 77, 1024),
                                   (1, 50280, 2560), (2, 300, 5120), (3, 40000, 544), (4, 20000, 2560), (4, 100, 8224), (5, 1000, 2560), (9, 5000, 2080), (16, 50280, 1536)])
def test_linear_is_the_product_of_quantised_rows(dev, dtype, m, n, k):
    torch.manual_seed(m + n + k)
    x = (torch.randn(m, k) * (1 + 9 * (torch.rand(k) < 0.05))).to(TYPES[dtype]).to(dev)
    w, w_scales = ops.mxfp4_quant(torch.randn(n, k, device=dev))
    codes, scales = ops.mxfp4_quant(x)
    for out in (None, torch.float16, torch.bfloat16, torch.float32):
        got = ops.mxfp4_linear(x, w, w_scales, out)
        assert got.dtype == (out or x.dtype)
        assert torch.equal(got, ops.mxfp4_mm(codes, scales, w, w_scales, got.dtype))
    # rows apart, on any address; dimensions in front
    wide = torch.zeros(m, k + 3, dtype=x.dtype, device=dev)
    wide[:, 1:k + 1] = x
    assert torch.equal(ops.mxfp4_linear(wide[:, 1:k + 1], w, w_scales), ops.mxfp4_linear(x, w, w_scales))
    assert torch.equal(ops.mxfp4_linear(x.view(1, m, 1, k), w, w_scales), ops.mxfp4_linear(x, w, w_scales).view(1, m, 1, n))


@pytest.mark.parametrize("m", [1, 16, 40, 150, 400])
def test_nan_stays_in_its_row_or_column(dev, m):
    n, k = 300, 1056
    g = np.random.default_rng(m)
    a, a_scales, w, w_scales, want = exact_case(g, m, n, k, dev)
    a_nat, w_nat = ops.mxfp4_scales_of(a_scales, 33), ops.mxfp4_scales_of(w_scales, 33)
    a_nat[m // 2, 32] = 255
    w_nat[17, 0] = 255
    w_nat[299, 20] = 255
    got = ops.mxfp4_mm(a, ops.mxfp4_scales(a_nat), w, ops.mxfp4_scales(w_nat), torch.float32).cpu()
    lost = torch.zeros(m, n, dtype=torch.bool)
    lost[m // 2], lost[:, 17], lost[:, 299] = True, True, True
    assert torch.equal(got.isnan(), lost) and torch.equal(got[~lost], want.float()[~lost])


@pytest.mark.parametrize("m", [1, 30, 70, 150, 400])
def test_bytes_behind_the_last_block_are_not_looked_at(dev, m):
    n, k = 200, 1056                                               # two groups and a block
    a, a_scales, w, w_scales, want = exact_case(np.random.default_rng(m), m, n, k, dev)
    for s in (a_scales, w_scales):
        behind = torch.ones(16, dtype=torch.bool)
        behind[0] = False
        s[2, :, behind] = 255
    assert torch.equal(ops.mxfp4_mm(a, a_scales, w, w_scales, torch.float32).cpu(), want.float())
    assert torch.equal(ops.mxfp4_dequant(a, a_scales), ops.mxfp4_dequant(a, a_scales.masked_fill(a_scales == 255, 0)))


@pytest.mark.parametrize("m", [1, 20, 80, 300])
def test_operands_as_they_lie(dev, m):
    """rows of codes apart, parts of larger operands; the scales of those"""
    n, k = 150, 1152
    a, a_scales, w, w_scales, want = exact_case(np.random.default_rng(m), m + 5, n + 9, k, dev)
    apart = torch.full((m + 5, k // 2 + 48), 0x77, dtype=torch.uint8, device=dev)
    apart[:, 32:32 + k // 2] = a
    got = ops.mxfp4_mm(apart[3:3 + m, 32:32 + k // 2], a_scales[:, 3:3 + m], w[7:7 + n], w_scales[:, 7:7 + n], torch.float32)
    assert torch.equal(got.cpu(), want[3:3 + m, 7:7 + n].float())


@pytest.mark.parametrize("scale", [0, 100, 254])
def test_scales_at_either_end(dev, scale):
    """products of 2^-127 by 2^127 and the like; what passes fp32 is infinite, what falls below it nothing"""
    n, k = 40, 64
    g = np.random.default_rng(scale)
    for m in (3, 40, 200):
        codes = g.integers(0, 16, (m, k)).astype(np.uint8)
        a, a_scales, a_values = operand(g, m, k, 0, 0, dev)
        w, w_scales, w_values = operand(g, n, k, 0, 0, dev)
        for other in (254 - scale, 254, 0):
            a_s, w_s = torch.full_like(a_scales, scale), torch.full_like(w_scales, other)
            with np.errstate(over="ignore"):
                want = ((a_values @ w_values.T) * 2.0 ** (scale - 127) * 2.0 ** (other - 127)).astype(np.float32)
            got = ops.mxfp4_mm(a, a_s, w, w_s, torch.float32).cpu().numpy()
            # (where the magnitudes' sum passes fp32 a product or a partial sum may: 2^127 by 2^127 does, also where all of them cancel)
            with np.errstate(over="ignore"):
                size = (np.abs(a_values) @ np.abs(w_values).T) * 2.0 ** (scale - 127) * 2.0 ** (other - 127)
            big = size >= np.finfo(np.float32).max / 8
            small = ~big & (np.abs(want) < np.finfo(np.float32).tiny * (64 * 36))      # (and a product may fall below it)
            assert np.array_equal(got[~big & ~small], want[~big & ~small]) and np.all(np.abs(got[small]) <= np.finfo(np.float32).tiny * (64 * 64 * 36))


def test_nothing(dev):
    w, w_scales = ops.mxfp4_quant(torch.zeros(5, 64, device=dev))
    assert ops.mxfp4_linear(torch.zeros(0, 64, device=dev), w, w_scales).shape == (0, 5)
    assert ops.mxfp4_linear(torch.zeros(2, 0, 64, device=dev), w, w_scales).shape == (2, 0, 5)
    assert ops.mxfp4_mm(w[:0], w_scales[:, :0], w, w_scales).shape == (0, 5)
    assert ops.mxfp4_mm(w, w_scales, w[:0], w_scales[:, :0]).shape == (5, 0)
    empty = ops.mxfp4_quant(torch.zeros(3, 0, device=dev))
    got = ops.mxfp4_mm(*empty, *ops.mxfp4_quant(torch.zeros(4, 0, device=dev)))
    assert got.shape == (3, 4) and not got.any()


def test_refusals(dev):
    a, a_scales = ops.mxfp4_quant(torch.zeros(4, 64, device=dev))
    w, w_scales = ops.mxfp4_quant(torch.zeros(6, 64, device=dev))
    other, other_scales = ops.mxfp4_quant(torch.zeros(6, 96, device=dev))
    x = torch.zeros(4, 64, device=dev)
    for args in ((a, a_scales, other, other_scales), (a, w_scales, w, w_scales), (a, a_scales, w, a_scales), (a.int(), a_scales, w, w_scales), (a[0], a_scales, w, w_scales),
                 (a, a_scales, w.cpu(), w_scales), (a, a_scales, w, w_scales.cpu()), (a.t(), a_scales, w, w_scales)):
        with pytest.raises(RuntimeError):
            ops.mxfp4_mm(*args)
    for args in ((x[:, :32], w, w_scales), (x.int(), w, w_scales), (x.cpu(), w, w_scales), (x.double(), w, w_scales)):
        with pytest.raises(RuntimeError):
            ops.mxfp4_linear(*args)
    with pytest.raises(NotImplementedError):
        ops.mxfp4_mm(a, a_scales, w, w_scales, torch.int8)
    with pytest.raises(NotImplementedError):
        ops.mxfp4_linear(x, w, w_scales, torch.float64)


@pytest.mark.parametrize("m", [1, 50, 300])
def test_captured(dev, m):
    """two graphs, each with workspace of its own, replayed in turn with eager calls between them"""
    torch.manual_seed(m)
    w, w_scales = ops.mxfp4_quant(torch.randn(600, 1024, device=dev))
    xs = [torch.randn(m, 1024, device=dev).half() for _ in range(2)]
    ops.mxfp4_linear(xs[0], w, w_scales)
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.mxfp4_linear(x, w, w_scales))
        graphs.append(graph)
    for step in range(3):
        for x in xs:
            x.copy_(torch.randn(m, 1024, device=dev).half())
        want = [ops.mxfp4_linear(x, w, w_scales) for x in xs]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), step


def test_on_another_stream(dev):
    x = torch.randn(40, 512, device=dev)
    w, w_scales = ops.mxfp4_quant(torch.randn(300, 512, device=dev))
    want = ops.mxfp4_linear(x, w, w_scales)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.mxfp4_linear(x, w, w_scales)
    side.synchronize()
    assert torch.equal(got, want)


def test_module(dev):
    torch.manual_seed(1)
    layer = torch.nn.Linear(192, 77, bias=False).half().to(dev)
    q = MXFP4Linear.from_fp16(layer)
    x = torch.randn(2, 5, 192, device=dev).half()
    assert torch.equal(q(x), ops.mxfp4_linear(x, q.weight, q.weight_scales))
    codes, scales = ops.mxfp4_quant(x)
    assert torch.equal(q(codes, scales), q(x))
    assert torch.equal(q.dequantized_weight(), ops.mxfp4_dequant(*ops.mxfp4_quant(layer.weight)))
    other = MXFP4Linear(192, 77, device=dev, out_dtype=torch.float32)
    other.load_state_dict(q.state_dict())
    assert other(x).dtype == torch.float32 and torch.equal(other(x).half(), q(x))
    tokens = torch.randint(0, 77, (2, 5), device=dev)
    assert all(torch.equal(a, b) for a, b in zip(q.token_logprobs(x, tokens, 3), ops.token_logprobs(q(x), tokens, 3)))
    with pytest.raises(AssertionError):
        MXFP4Linear.from_fp16(torch.nn.Linear(64, 8).to(dev))
    with pytest.raises(AssertionError):
        MXFP4Linear(40, 8, device=dev)


@pytest.mark.parametrize("m,n,k,linear,names", [
    (1, 100, 64, False, ["mxfp4_direct_kernel<1, 1, signed char, false>"]), (1, 60000, 64, False, ["mxfp4_tiles_kernel<1, 2, 2, 4, 3, true>"]),
    (17, 4000, 512, False, ["mxfp4_direct_kernel<2, 1, signed char, false>"]), (20, 6000, 512, False, ["mxfp4_direct_kernel<2, 2, signed char, false>"]),
    (64, 4000, 512, False, ["mxfp4_direct_kernel<2, 2, signed char, false>"]), (64, 8000, 512, False, ["mxfp4_direct_kernel<4, 2, signed char, false>"]),
    (1, 40000, 96, True, ["mxfp4_direct_kernel<1, 1, float, true>"]), (9, 700, 1056, True, ["mxfp4_direct_kernel<1, 1, float, false>"]),
    (16, 60000, 96, True, ["mxfp4_quant_kernel<", "mxfp4_tiles_kernel<1, 2, 2, 4, 3, true>"]), (17, 4000, 512, True, ["mxfp4_quant_kernel<", "mxfp4_direct_kernel<2, 1, signed char, false>"]),
    (100, 9000, 512, False, ["mxfp4_tiles_kernel<1, 2, 2, 2, 4, false>"]), (300, 9000, 96, False, ["mxfp4_tiles_kernel<2, 1, 2, 4, 4, true>"]),
    (300, 20000, 512, False, ["mxfp4_tiles_kernel<2, 2, 2, 4, 3, false>"]), (4000, 9000, 512, False, ["mxfp4_stream_kernel", "mxfp4_tiles_kernel<2, 1, 2, 4, 4, false>"]),
    (4300, 9000, 96, False, ["mxfp4_tiles_kernel<4, 2, 2, 4, 2, true>", "mxfp4_tiles_kernel<2, 2, 2, 4, 3, true>"])])
def test_the_choice_of_kernels(dev, m, n, k, linear, names):
    g = np.random.default_rng(m)
    w, w_scales, _ = operand(g, n, k, 0, 2, dev)
    if linear:
        x = torch.randn(m, k, device=dev)
        expect(kernels(lambda: ops.mxfp4_linear(x, w, w_scales))[1], *names)
    else:
        a, a_scales, _ = operand(g, m, k, 0, 2, dev)
        expect(kernels(lambda: ops.mxfp4_mm(a, a_scales, w, w_scales))[1], *names)


@pytest.mark.parametrize("m,n", [(70001, 40003), (2200000, 1001), (15, 150000000), (3, 900000000)])
def test_offsets_past_32_bits(dev, m, n):
    """outputs of more than 2^31 numbers or operands of more than 2 GiB"""
    k = 32 if n < 1 << 24 else 64
    def big(rows, generator):
        few = min(rows, 997)                               # (row r is row r % few of these)
        codes, scales, values = operand(generator, few, k, 0, 2, dev)
        times = -(-rows // few)
        return codes.repeat(times, 1)[:rows], scales.repeat(1, times, 1)[:, :rows].contiguous(), torch.from_numpy(values).to(dev), few
    g = np.random.default_rng(m)
    a, a_scales, a_values, of_a = big(m, g)
    w, w_scales, w_values, of_w = big(n, g)
    got = ops.mxfp4_mm(a, a_scales, w, w_scales, torch.bfloat16)
    want = (a_values @ w_values.T).float().bfloat16()
    rows = torch.tensor(sorted({0, 1 % m, m // 2, m - 2 if m > 1 else 0, m - 1}), device=dev)
    for r in rows.tolist():
        row = want[r % of_a]
        for first in range(0, n, 1 << 27):
            last = min(n, first + (1 << 27))
            at = torch.arange(first, last, device=dev) % of_w
            assert torch.equal(got[r, first:last], row[at]), (r, first)


def test_a_small_layer_is_saved_by_itself(dev, tmp_path):
    """weights and scales in memory of their own each, whatever mxfp4_quant does with small answers"""
    q = MXFP4Linear.from_fp16(torch.nn.Linear(64, 8, bias=False).half().to(dev))
    assert q.weight.untyped_storage().data_ptr() != q.weight_scales.untyped_storage().data_ptr()
    checkpoints = pytest.importorskip("safetensors.torch")
    checkpoints.save_model(q, str(tmp_path / "layer.safetensors"))
    other = MXFP4Linear(64, 8, device=dev)
    checkpoints.load_model(other, str(tmp_path / "layer.safetensors"))
    x = torch.randn(3, 64, device=dev).half()
    assert torch.equal(other(x), q(x))
