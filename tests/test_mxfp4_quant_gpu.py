"""Microscaled 4-bit floating point: codes, scales and values against the definition, bit for bit."""
import numpy as np
import pytest
import torch

from mxfp4_reference import packed, quantised, unpacked, values_of
from quamba_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def check(x):
    """x (rows, K) on the GPU"""
    rows, k = x.shape
    codes, scales = ops.mxfp4_quant(x)
    assert codes.shape == (rows, k // 2) and codes.dtype == torch.uint8 and scales.shape == (-(-k // 512), rows, 16) and scales.dtype == torch.uint8
    want_codes, want_scales, want = quantised(x.cpu().double().numpy())
    assert torch.equal(scales.cpu(), ops.mxfp4_scales(torch.from_numpy(want_scales)))            # (zeros behind the last block among them)
    fine = np.repeat(want_scales != 255, 32, 1)
    assert np.array_equal(unpacked(codes)[fine], want_codes[fine])
    for dtype in TYPES.values():
        got = ops.mxfp4_dequant(codes, scales, dtype)
        assert got.dtype == dtype and torch.equal(got.cpu().nan_to_num(7.0), torch.from_numpy(want).to(dtype).nan_to_num(7.0)) and torch.equal(
            got.cpu().isnan(), torch.from_numpy(np.isnan(want)))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 768), (3, 64), (2, 480), (5, 512), (17, 544), (100, 96), (4, 1056), (33, 2560), (7, 5120)])
def test_sizes(dev, dtype, rows, k):
    g = torch.Generator().manual_seed(rows * k)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-8, 9, (rows, k), generator=g).float())
    check(x.to(TYPES[dtype]).to(dev))


@pytest.mark.parametrize("dtype,bits", [("fp16", torch.int16), ("bf16", torch.int16)])
def test_every_16_bit_number(dev, dtype, bits):
    """next to others of its size and to any others, infinities and NaNs among them"""
    every = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(bits)
    mixed = every[torch.randperm(1 << 16, generator=torch.Generator().manual_seed(3))]
    for order in (every, mixed):
        check(order.view(TYPES[dtype]).view(-1, 64).to(dev))
    # and with no more than one block in a hundred lost to them
    finite = mixed.view(TYPES[dtype])
    finite = torch.where(finite.isfinite(), finite, torch.zeros_like(finite))
    check(finite.view(-1, 64).to(dev))


def test_borders(dev):
    """of 32 bits: what lies on a border between two values and one step to either side, at every size there is"""
    rows = []
    for e in list(range(-151, 128)):
        s = 2.0 ** max(e - 2, -127)
        borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]) * s
        with np.errstate(over="ignore"):
            row = np.concatenate([borders, np.nextafter(borders.astype(np.float32), np.float32(0)), np.nextafter(borders.astype(np.float32), np.float32(np.inf)), [4 * s] * 8]).astype(np.float32)
        rows.append(np.where(np.isfinite(row), row, np.float32(1.0)))
    x = torch.from_numpy(np.array(rows))
    check(torch.cat((x, -x)).to(dev))


def test_blocks_that_are_nan(dev):
    x = torch.randn(6, 96)
    x[0, 3], x[1, 40], x[2, 95], x[3, 0] = float("nan"), float("inf"), float("-inf"), -float("nan")
    check(x.to(dev))
    codes, scales = ops.mxfp4_quant(x.to(dev))
    natural = ops.mxfp4_scales_of(scales, 3).cpu()
    assert (natural == 255).sum() == 4 and natural[4:].max() < 255


def test_zeros_and_the_smallest(dev):
    x = torch.zeros(3, 64)
    x[1, 0] = -0.0
    x[2, :3] = torch.tensor([2.0 ** -149, 2.0 ** -128, -(2.0 ** -127)])
    check(x.to(dev))
    codes, scales = ops.mxfp4_quant(x.to(dev))
    assert int(scales.max()) == 0 and int(codes[0].max()) == 0


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_rows_as_they_lie(dev, dtype):
    """rows apart, on addresses of any number, in dimensions in front"""
    base = torch.randn(9, 1200, device=dev).to(TYPES[dtype])
    for x in (base[:, 1:1025], base[::2, 3:547], base[2:, 8:520], base[:1, 5:37]):
        assert not x.is_contiguous() or x.shape[0] == 1
        got, want = ops.mxfp4_quant(x), ops.mxfp4_quant(x.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(4, 3, 5, 64, device=dev).to(TYPES[dtype])
    for y in (x, x.transpose(0, 1), x[:, :, ::2], x[0, 0, 0]):
        codes, scales = ops.mxfp4_quant(y)
        assert codes.shape == (*y.shape[:-1], 32)
        flat = ops.mxfp4_quant(y.reshape(-1, 64))
        assert torch.equal(codes.reshape(-1, 32), flat[0]) and torch.equal(scales, flat[1])
        assert ops.mxfp4_dequant(codes, scales).shape == y.shape


def test_nothing(dev):
    for shape in ((0, 64), (3, 0), (2, 0, 96)):
        codes, scales = ops.mxfp4_quant(torch.zeros(shape, device=dev))
        assert codes.shape == (*shape[:-1], shape[-1] // 2)
        assert ops.mxfp4_dequant(codes, scales, torch.float16).shape == shape


def test_dequant_of_rows_as_they_lie(dev):
    g = np.random.default_rng(5)
    codes = g.integers(0, 16, (6, 1088)).astype(np.uint8)
    scales = g.integers(0, 256, (6, 34)).astype(np.uint8)
    laid = torch.full((4, 9, 16), 255, dtype=torch.uint8, device=dev)
    laid[:3, 3:] = ops.mxfp4_scales(torch.from_numpy(scales)).to(dev)
    apart = torch.zeros(6, 640, dtype=torch.uint8, device=dev)
    apart[:, 16:560] = packed(codes).to(dev)
    want = torch.from_numpy(values_of(codes, scales))
    for dtype in TYPES.values():
        got = ops.mxfp4_dequant(apart[:, 16:560], laid[:3, 3:], dtype).cpu()
        assert torch.equal(got.nan_to_num(7.0), want.to(torch.float32).to(dtype).nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())


def test_refusals(dev):
    x = torch.zeros(4, 64, device=dev)
    codes, scales = ops.mxfp4_quant(x)
    for bad in (x[:, :33], x.int(), x.t(), x[0, 0], x.double(), x.cpu(), x.expand(2, 4, 64).reshape(8, 64).as_strided((8, 64), (32, 1))):
        with pytest.raises(RuntimeError):
            ops.mxfp4_quant(bad)
    big = torch.zeros(4, 72, dtype=torch.uint8, device=dev)
    for c, s in ((codes[:, :24], scales), (codes.int(), scales), (codes, scales[:, :3]), (codes, scales.cpu()), (codes, scales.int()), (codes, scales[0]),
                 (codes, scales.transpose(0, 1)), (big[:, 8:40], scales), (big[:, :32], scales), (codes, torch.zeros(1, 4, 32, dtype=torch.uint8, device=dev)[..., ::2]),
                 (codes, torch.zeros(65 + 8, dtype=torch.uint8, device=dev)[8:72].view(1, 4, 16))):
        with pytest.raises(RuntimeError):
            ops.mxfp4_dequant(c, s)
    with pytest.raises(NotImplementedError):
        ops.mxfp4_dequant(codes, scales, torch.float64)


def test_captured_and_on_another_stream(dev):
    x = torch.randn(40, 1056, device=dev)
    ops.mxfp4_dequant(*ops.mxfp4_quant(x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scales = ops.mxfp4_quant(x)
        values = ops.mxfp4_dequant(codes, scales, torch.bfloat16)
    for step in range(3):
        x.copy_(torch.randn(40, 1056, device=dev) * 10.0 ** step)
        want = (*ops.mxfp4_quant(x), ops.mxfp4_dequant(*ops.mxfp4_quant(x), torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((codes, scales, values), want)), step
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.mxfp4_quant(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits(dev):
    """rows more than 4 GiB into numbers, and 2 GiB into codes"""
    rows, k = 2100000, 2048
    x = torch.zeros(rows, k, dtype=torch.float16, device=dev)
    some = [0, 1, 524287, 524288, 1048577, rows - 9, rows - 1]
    x[some] = torch.randn(len(some), k, generator=torch.Generator().manual_seed(1)).half().to(dev)
    codes, scales = ops.mxfp4_quant(x)
    want_codes, want_scales = ops.mxfp4_quant(x[some])
    assert torch.equal(codes[some], want_codes) and torch.equal(scales[:, some], want_scales)
    values = ops.mxfp4_dequant(codes, scales, torch.float16)
    assert torch.equal(values[some], ops.mxfp4_dequant(want_codes, want_scales, torch.float16)) and int(values.count_nonzero(1).count_nonzero()) == len(some)
