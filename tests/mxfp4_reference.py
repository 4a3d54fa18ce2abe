"""Microscaled 4-bit floating point in numpy's 64 bits, from its definition (test helper)."""
import numpy as np
import torch

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantised(x):
    """(codes (rows, K), scale bytes (rows, K / 32), values (rows, K)) of rows in 64 bits; codes of a block that is NaN are 0."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    most = np.abs(b).max(-1)
    e = np.maximum(np.where(most > 0, np.floor(np.log2(np.where(most > 0, most, 1.0))), -1000) - 2, -127)
    # (log2 rounds next to a power of two)
    e = np.where(most >= np.exp2(e + 3), e + 1, e)
    e = np.where((most < np.exp2(e + 2)) & (e > -127), e - 1, e)
    ratio = np.abs(b) * np.exp2(-e)[..., None]
    off = np.abs(ratio[..., None] - VALUES)
    codes = np.argmin(off + 1e-9 * (np.arange(8) % 2), -1)                # (of two as near the even one; others differ by far more than that)
    near = np.sort(off, -1)
    tie = near[..., 0] == near[..., 1]
    codes = np.where(tie, np.argmin(off, -1) + np.argmin(off, -1) % 2, codes)
    values = np.copysign(VALUES[codes], b) * np.exp2(e)[..., None]
    values = np.where(bad[..., None], np.nan, values).reshape(rows, k)
    codes = (codes + 8 * np.signbit(b)).reshape(rows, k)
    return codes.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8), values


def values_of(codes, scales):
    """Of codes (rows, K) and scale bytes (rows, K / 32)."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, 1)


def packed(codes):
    return torch.from_numpy((codes[:, ::2] | codes[:, 1::2] << 4).astype(np.uint8))


def unpacked(t):
    t = t.cpu().numpy()
    out = np.empty((t.shape[0], 2 * t.shape[1]), np.uint8)
    out[:, ::2], out[:, 1::2] = t & 15, t >> 4
    return out


def operand(g, rows, k, low, high, dev):
    """Random codes, scales of 2^low .. 2^high: (codes uint8 (rows, k / 2), scales as mxfp4_quant lays them out, values in 64 bits)."""
    from quamba_amd import ops
    codes = g.integers(0, 16, (rows, k)).astype(np.uint8)
    scales = g.integers(127 + low, 128 + high, (rows, k // 32)).astype(np.uint8)
    return packed(codes).to(dev), ops.mxfp4_scales(torch.from_numpy(scales)).to(dev), values_of(codes, scales)
