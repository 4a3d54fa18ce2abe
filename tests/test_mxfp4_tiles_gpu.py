"""Products of microscaled 4-bit operands in tiles, each kernel by name together with what it gives: K of several groups of scales, whole ones or not, an even or odd number of k tiles.

Sums are exact, or bounded, as in test_mxfp4_mm_gpu.py.  Operands repeat 997 rows, a prime that no tile's size divides: tiles that change places show."""
import numpy as np
import pytest
import torch

from launched import expect, kernels
from mxfp4_reference import operand
from quamba_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# m, n, k, the first kernel (256 CUs); k 1056 is 2 groups and a block in 5 k tiles, 1312 2.6 groups in 6, 1568 3 groups and a block in 7, 2560 5 groups in 10
KERNELS = [
    (100, 9000, 1056, "mxfp4_tiles_kernel<1, 2, 2, 2, 4, true>"), (65, 11003, 1568, "mxfp4_tiles_kernel<1, 2, 2, 2, 4, true>"), (128, 9000, 2560, "mxfp4_tiles_kernel<1, 2, 2, 2, 4, false>"),
    (17, 60000, 1056, "mxfp4_tiles_kernel<1, 2, 2, 4, 3, true>"), (33, 40001, 1312, "mxfp4_tiles_kernel<1, 2, 2, 4, 3, true>"), (64, 50280, 2560, "mxfp4_tiles_kernel<1, 2, 2, 4, 3, false>"),
    (300, 9000, 1056, "mxfp4_tiles_kernel<2, 1, 2, 4, 4, true>"), (270, 9001, 1568, "mxfp4_tiles_kernel<2, 1, 2, 4, 4, true>"), (384, 9000, 1536, "mxfp4_tiles_kernel<2, 1, 2, 4, 4, false>"),
    (300, 20000, 1568, "mxfp4_tiles_kernel<2, 2, 2, 4, 3, true>"), (257, 20003, 1056, "mxfp4_tiles_kernel<2, 2, 2, 4, 3, true>"), (384, 20000, 2560, "mxfp4_tiles_kernel<2, 2, 2, 4, 3, false>"),
    (4300, 9000, 1056, "mxfp4_tiles_kernel<4, 2, 2, 4, 2, true>"), (4000, 4001, 1568, "mxfp4_tiles_kernel<4, 2, 2, 4, 2, true>"), (4096, 4096, 1536, "mxfp4_tiles_kernel<4, 2, 2, 4, 2, false>"),
    (700, 50001, 1536, "mxfp4_stream_kernel"), (4000, 9000, 2560, "mxfp4_stream_kernel")]
MASKED = [c for c in KERNELS if c[2] % 512]
FEW = [KERNELS[i] for i in (1, 4, 7, 10, 12, 15)]


def repeated(g, rows, k, low, high, dev):
    """(codes, scales, values in 64 bits on the GPU)"""
    few = min(rows, 997)
    codes, scales, values = operand(g, few, k, low, high, dev)
    times = -(-rows // few)
    return codes.repeat(times, 1)[:rows], scales.repeat(1, times, 1)[:, :rows].contiguous(), torch.from_numpy(values).to(dev).repeat(times, 1)[:rows]


def both(m, n, k, dev, low=0, high=2):
    g = np.random.default_rng(m + n + k)
    return repeated(g, m, k, low, high, dev), repeated(g, n, k, low, high, dev)


def product(a, w, dtype, name):
    torch.cuda.synchronize()
    got, names = kernels(lambda: ops.mxfp4_mm(*a[:2], *w[:2], dtype))
    expect(names, name)
    return got


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_exact_sums(dev, m, n, k, name):
    a, w = both(m, n, k, dev)
    want = (a[2] @ w[2].T).float()
    for dtype in TYPES.values():
        assert torch.equal(product(a, w, dtype, name), want.to(dtype)), dtype


@pytest.mark.parametrize("m,n,k,name", FEW)
def test_sums_that_round(dev, m, n, k, name):
    a, w = both(m, n, k, dev, -12, 12)
    want, size = a[2] @ w[2].T, a[2].abs() @ w[2].abs().T
    instructions = (k + 127) // 128
    for dtype in (torch.float32, torch.bfloat16):
        half = torch.finfo(dtype).eps / 2
        off = (product(a, w, dtype, name).double() - want).abs()
        assert (off <= size * (2.0 ** -18 * instructions + 2.0 ** -24 * 16) * (1 + half) + want.abs() * half).all()
        assert off.mean() <= (size * 2.0 ** -24 * instructions + want.abs() * half).mean()


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_nan_stays_in_its_row_or_column(dev, m, n, k, name):
    a, w = both(m, n, k, dev)
    blocks = k // 32
    a_nat, w_nat = ops.mxfp4_scales_of(a[1], blocks).clone(), ops.mxfp4_scales_of(w[1], blocks).clone()
    a_nat[m // 2, blocks - 1], a_nat[m - 1, 17] = 255, 255
    w_nat[17, 0], w_nat[n // 3, 20], w_nat[n - 1, blocks - 1] = 255, 255, 255
    got = product((a[0], ops.mxfp4_scales(a_nat)), (w[0], ops.mxfp4_scales(w_nat)), torch.float32, name)
    lost = torch.zeros(m, n, dtype=torch.bool, device=dev)
    lost[m // 2], lost[m - 1], lost[:, 17], lost[:, n // 3], lost[:, n - 1] = True, True, True, True, True
    assert torch.equal(got.isnan(), lost) and torch.equal(got[~lost], (a[2] @ w[2].T).float()[~lost])


@pytest.mark.parametrize("m,n,k,name", MASKED)
def test_bytes_behind_the_last_block_are_not_looked_at(dev, m, n, k, name):
    a, w = both(m, n, k, dev)
    behind = torch.tensor([16 * (k // 512) + 4 * (place % 4) + place // 4 >= k // 32 for place in range(16)])
    assert behind.any()
    for s in (a[1], w[1]):
        s[-1, :, behind] = 255
    assert torch.equal(product(a, w, torch.float32, name), (a[2] @ w[2].T).float())


@pytest.mark.parametrize("m,n,k,name", FEW + KERNELS[-1:])
def test_operands_as_they_lie(dev, m, n, k, name):
    """rows of codes apart, parts of larger operands; the scales of those"""
    a, w = both(m + 5, n + 9, k, dev)
    apart = [torch.full((t.shape[0], k // 2 + 48), 0x77, dtype=torch.uint8, device=dev) for t in (a[0], w[0])]
    for to, (codes, *_) in zip(apart, (a, w)):
        to[:, 32:32 + k // 2] = codes
    got = product((apart[0][3:3 + m, 32:32 + k // 2], a[1][:, 3:3 + m]), (apart[1][7:7 + n, 32:32 + k // 2], w[1][:, 7:7 + n]), torch.float32, name)
    assert torch.equal(got, (a[2][3:3 + m] @ w[2][7:7 + n].T).float())


@pytest.mark.parametrize("m,n,k,name", FEW)
@pytest.mark.parametrize("low", [0, 100, 254])
def test_scales_at_either_end(dev, m, n, k, name, low):
    """products of 2^-127 by 2^127 and the like"""
    a, w = both(m, n, k, dev, 0, 0)
    got = product((a[0], torch.full_like(a[1], low)), (w[0], torch.full_like(w[1], 254 - low)), torch.float32, name)
    assert torch.equal(got, (a[2] @ w[2].T).float())


@pytest.mark.parametrize("m,n,k,name", FEW)
def test_captured(dev, m, n, k, name):
    """replayed after other operands came to the same places, with eager calls between"""
    a, w = both(m, n, k, dev)
    product(a, w, torch.float16, name)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.mxfp4_mm(*a[:2], *w[:2])
    for step in range(3):
        a[0].copy_(a[0].roll(1, 0))
        w[0].copy_(w[0].roll(3, 0))
        want = ops.mxfp4_mm(*a[:2], *w[:2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step


def test_rows_of_numbers_in_front_of_tiles(dev):
    """mxfp4_linear of many rows: quantisation, then tiles, the bits of both by themselves, and the product itself against the values"""
    for m, n, k, name in FEW:
        torch.manual_seed(m)
        x = (torch.randn(m, k, device=dev) * (1 + 9 * (torch.rand(k, device=dev) < 0.05))).half()
        w = repeated(np.random.default_rng(n), n, k, -2, 2, dev)
        torch.cuda.synchronize()
        got, names = kernels(lambda: ops.mxfp4_linear(x, *w[:2], torch.float32))
        expect(names, name)
        codes, scales = ops.mxfp4_quant(x)
        assert torch.equal(got, ops.mxfp4_mm(codes, scales, *w[:2], torch.float32))
        values = ops.mxfp4_dequant(codes, scales).double()
        want, size = values @ w[2].T, values.abs() @ w[2].abs().T
        assert ((got.double() - want).abs() <= size * (2.0 ** -18 * ((k + 127) // 128) + 2.0 ** -24 * 17) + want.abs() * 2.0 ** -24).all()
