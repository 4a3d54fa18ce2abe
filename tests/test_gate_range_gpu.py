"""The gate of add_rmsnorm over its whole range, against 64 bits.

sigmoid(z) = 1 / (1 + 2^(-z log2 e)) in fp32, units of 2^-24: the exponent's product and the rounding of log2 e 1.22 |z|, the exponential and the
reciprocal 2 each, the sum 1; the products with z, with x and with the scale 1 each: 8 + 1.25 |z|.  Below z = -87.3 the reciprocal is no normal number any more
and may be 0: off by at most 2^-126 |x| max(1, |z|), twice that with its roundings."""
import numpy as np
import pytest
import torch

from quamba_amd import ops
from test_add_rmsnorm_gpu import TYPES, call, make, want_of
from test_add_rmsnorm_gpu import check as check_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
VALUES = [0.0, 1.0, 5.0, 20.0, 60.0, 86.0, 87.0, 87.5, 88.0, 89.0, 90.0, 103.0, 104.0, 1000.0, 60000.0]


def _gate(dim, rows):
    v = torch.tensor([s * x for x in VALUES for s in (1, -1)])
    return torch.stack([v.roll(i).repeat(-(-dim // len(v)))[:dim] for i in range(rows)])


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 1000, 4099])
def test_gates_alone(dev, dtype, act, dim):
    a = make(4, dim, TYPES[dtype], dev, residual=None)
    gate = _gate(dim, 4).to(TYPES[dtype]).to(dev)
    v = ops.add_rmsnorm(a["x"], a["weight"], 1e-5, gate=gate, gate_act=act, residual_dtype=torch.float32)[1].cpu().double().numpy()
    x, z = a["x"].cpu().double().numpy(), gate.cpu().double().numpy()
    with np.errstate(over="ignore"):
        want = x * (z if act == "silu" else 1.0) / (1 + np.exp(-z))
    assert np.all(np.abs(v - want) <= (8 + 1.25 * np.abs(z)) * U * np.abs(want) + 2.0 ** -125 * np.abs(x) * np.maximum(1, np.abs(z)))


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_gates_in_front_of_the_sum(dev, dtype, act):
    """the bounds of the operator's own test hold to |z| of 100: 8 + 1.25 |z| units are within its 256 (beyond, sigmoid is 1 to within a unit, or 0)"""
    for dim in (512, 1531):
        a = make(5, dim, TYPES[dtype], dev, residual="fp32", post=True, gate=("rows", act))
        a["gate"] = _gate(dim, 5).clamp(-1000, 1000).to(TYPES[dtype]).to(dev)
        with np.errstate(over="ignore"):
            want = want_of(a)
        check_norm(call(a), want, a["x"])
        check_norm(call(a, out_dtype=torch.int8), want, a["x"])
