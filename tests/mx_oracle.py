"""Microscaled 4-bit formats in 64 bits on the CPU (numpy): what the operators of
include/gemmzoo/microscale.h are defined to compute.  Test infrastructure only."""
from __future__ import annotations

import math

import numpy as np

FP4, NVFP4 = 16, 17
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([MAGNITUDES, -MAGNITUDES])
BORDERS = (MAGNITUDES[1:] + MAGNITUDES[:-1]) / 2  # 0.25 0.75 1.25 1.75 2.5 3.5 5
E4M3 = np.array([(m * 2.0 ** -9) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)])[:127]


def block(fmt):
    return 16 if fmt == NVFP4 else 32


def scale_values(b, fmt):
    b = np.asarray(b, dtype=np.int64)
    if fmt == FP4:
        return np.where(b == 255, np.nan, np.ldexp(1.0, b - 127))
    return np.where(b >= 127, np.nan, E4M3[np.minimum(b, 126)])


def nearest_even(x, grid):
    """Index of the grid value nearest to x >= 0 (ties to the even index, beyond the end the last)."""
    i = np.clip(np.searchsorted(grid, x, side="right") - 1, 0, len(grid) - 1)
    j = np.minimum(i + 1, len(grid) - 1)
    lo, hi = x - grid[i], grid[j] - x
    up = (hi < lo) | ((hi == lo) & (i % 2 == 1))
    return np.where((j > i) & up, j, i)


def quantize(x, fmt):
    """(codes 0..15 rows x k, scale bytes rows x blocks) of float64 values."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    bs = block(fmt)
    nb = -(-k // bs)
    p = np.zeros((rows, nb * bs))
    p[:, :k] = x
    b = p.reshape(rows, nb, bs)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(axis=2)
    bad = ~np.isfinite(amax)
    amax = np.where(bad, 0.0, amax)
    if fmt == FP4:
        e = np.where(amax > 0, np.frexp(np.where(amax > 0, amax, 1.0))[1] - 1 - 2, -127)
        byte = np.clip(e, -127, 127) + 127
    else:
        byte = nearest_even(amax / 6.0, E4M3)
    s = scale_values(byte, fmt)
    y = np.divide(np.where(np.isfinite(b), b, 0.0), s[:, :, None], out=np.zeros_like(b), where=s[:, :, None] > 0)
    codes = nearest_even(np.abs(y), MAGNITUDES) + 8 * np.signbit(b)
    codes = np.where(bad[:, :, None], 0, codes).reshape(rows, nb * bs)[:, :k]
    return codes.astype(np.uint8), np.where(bad, 255 if fmt == FP4 else 127, byte).astype(np.uint8)


def decode(codes, scales, fmt):
    bs = block(fmt)
    s = np.repeat(scale_values(scales, fmt), bs, axis=1)[:, :codes.shape[1]]
    return VALUES[codes] * s


def pack(codes):
    """rows x k codes -> rows x pitch bytes."""
    rows, k = codes.shape
    p = np.zeros((rows, -(-k // 32) * 32), dtype=np.uint8)
    p[:, :k] = codes
    return p[:, 0::2] | (p[:, 1::2] << 4)


def unpack(packed, k):
    c = np.empty((packed.shape[0], packed.shape[1] * 2), dtype=np.uint8)
    c[:, 0::2], c[:, 1::2] = packed & 15, packed >> 4
    return c[:, :k]


def tile(scales):
    """rows x blocks -> the 512-byte tiles, byte by byte from the definition."""
    rows, nb = scales.shape
    groups = -(-nb // 4)
    out = np.zeros(-(-rows // 128) * groups * 512, dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[((r // 128) * groups + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4] = scales
    return out


def untile(flat, rows, nb):
    groups = -(-nb // 4)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return flat[((r // 128) * groups + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4]


def act(x, name):
    if name == "relu":
        return np.maximum(x, 0)
    if name == "silu":
        return x / (1 + np.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + np.vectorize(math.erf)(x / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x
