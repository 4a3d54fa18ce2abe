"""Products of microscaled 4-bit operands straight from memory, each shape of that kernel by name, with K that gives all eight waves more than one group (8224: 16 and a block) or some
of them none (1056): what test_mxfp4_tiles_gpu.py asks of the tiles."""
import pytest
import torch

import test_mxfp4_tiles_gpu as tiles
from launched import expect, kernels
from quamba_amd import ops

pytestmark = pytest.mark.gpu
KERNELS = [
    (1, 500, 8224, "mxfp4_direct_kernel<1, 1, signed char, false>"), (16, 20003, 1056, "mxfp4_direct_kernel<1, 1, signed char, false>"), (40, 1001, 8224, "mxfp4_direct_kernel<1, 1, signed char, false>"),
    (17, 4001, 8224, "mxfp4_direct_kernel<2, 1, signed char, false>"), (31, 3999, 1056, "mxfp4_direct_kernel<2, 1, signed char, false>"),
    (64, 4001, 8224, "mxfp4_direct_kernel<2, 2, signed char, false>"), (33, 8003, 1056, "mxfp4_direct_kernel<4, 2, signed char, false>"),
    (64, 8003, 8224, "mxfp4_direct_kernel<4, 2, signed char, false>"), (511, 640, 8224, "mxfp4_direct_kernel<4, 2, signed char, false>")]


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_exact_sums(dev, m, n, k, name):
    a, w = tiles.both(m, n, k, dev)
    assert (a[2].abs() @ w[2].abs().T).max() < 2 ** 22              # (multiples of 1 / 4 below that are exact in whatever order)
    tiles.test_exact_sums(dev, m, n, k, name)


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_sums_that_round(dev, m, n, k, name):
    tiles.test_sums_that_round(dev, m, n, k, name)


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_nan_stays_in_its_row_or_column(dev, m, n, k, name):
    tiles.test_nan_stays_in_its_row_or_column(dev, m, n, k, name)


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_bytes_behind_the_last_block_are_not_looked_at(dev, m, n, k, name):
    tiles.test_bytes_behind_the_last_block_are_not_looked_at(dev, m, n, k, name)


@pytest.mark.parametrize("m,n,k,name", KERNELS)
def test_operands_as_they_lie(dev, m, n, k, name):
    tiles.test_operands_as_they_lie(dev, m, n, k, name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,shared", [(1, 700, 8224, "true"), (4, 4001, 8224, "true"), (3, 50, 1056, "true"), (5, 700, 4064, "false"), (16, 300, 1056, "false"), (9, 1001, 3616, "false")])
def test_rows_of_numbers(dev, dtype, m, n, k, shared):
    """quantised on the way, the bits of the product of their codes; a block with a NaN or an infinity is its row's alone"""
    torch.manual_seed(m + k)
    x = (torch.randn(m, k, device=dev) * torch.exp2(torch.randint(-6, 7, (m, k // 32), device=dev)).repeat_interleave(32, 1)).to(dtype)
    w, w_scales = ops.mxfp4_quant(torch.randn(n, k, device=dev))
    for spoilt in (None, float("nan"), float("-inf")):
        if spoilt is not None:
            x[m // 2, k - 1] = spoilt
        if dtype == torch.float32:                                 # (the profiler gives the names of the 16-bit ones as the compiler has them)
            got, names = kernels(lambda: ops.mxfp4_linear(x, w, w_scales, torch.float32))
            expect(names, f"mxfp4_direct_kernel<1, 1, float, {shared}>")
            assert len(names) <= 1
        else:
            got = ops.mxfp4_linear(x, w, w_scales, torch.float32)
        want = ops.mxfp4_mm(*ops.mxfp4_quant(x), w, w_scales, torch.float32)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
        lost = torch.zeros(m, dtype=torch.bool, device=dev)
        lost[m // 2] = spoilt is not None
        assert torch.equal(got.isnan(), lost[:, None].expand(m, n))
