"""Microscaled (MX) rows in float64: quantisation, values, RMSNorm, the product with 4-bit weights and the gated MLP
input. A block is 32 consecutive elements of a row; its scale is 2^(s - 127) with the byte s (255: NaN); codes are e4m3
bytes, or e2m1 half bytes with the earlier element in the low half; scales lie as [ceil(cols / 128), rows, 4].

Everything follows the definitions element by element: code tables are built from the formats' fields, and a value takes
the nearest table entry, ties to the even code.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
LARGEST = {"e4m3": 448.0, "e2m1": 6.0}


def _table(exp_bits, man_bits, bias, count):
    out = []
    for c in range(count):
        e, m = c >> man_bits, c & ((1 << man_bits) - 1)
        out.append(m * 2.0 ** (1 - bias - man_bits) if e == 0 else (1 + m / 2 ** man_bits) * 2.0 ** (e - bias))
    return np.array(out)


#: magnitudes by code, the sign bit aside (e4m3's code 127 is NaN and not in it)
TABLE = {"e4m3": _table(4, 3, 7, 127), "e2m1": _table(2, 1, 1, 8)}
SIGN = {"e4m3": 128, "e2m1": 8}


def scale_exponents(x, fmt):
    """Per block the least n >= -126 with max|x| <= LARGEST * 2^n; x [rows, cols] finite."""
    a = np.abs(x.reshape(x.shape[0], -1, BLOCK)).max(-1)
    n = np.full(a.shape, -126, np.int64)
    while True:
        over = a > LARGEST[fmt] * np.exp2(n.astype(np.float64))
        if not over.any():
            return n
        n[over] += 1


def _nearest(v, fmt):
    """Codes (without sign) of magnitudes v <= LARGEST: the nearest, ties to the even code."""
    t = TABLE[fmt]
    hi = np.searchsorted(t, v).clip(0, len(t) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = v - t[lo], t[hi] - v
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def quantize(x, fmt):
    """(codes uint8, one to an element, scales uint8 [ceil(cols / 128), rows, 4]) of x [rows, cols]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    bad = ~np.isfinite(x.reshape(rows, -1, BLOCK)).all(-1)
    y = np.where(np.repeat(bad, BLOCK, 1), 0.0, x)
    n = scale_exponents(y, fmt)
    q = y / np.repeat(np.exp2(n.astype(np.float64)), BLOCK, 1)
    codes = _nearest(np.abs(q), fmt) + SIGN[fmt] * np.signbit(q)
    s = np.where(bad, 255, n + 127)
    full = np.zeros((rows, -(-cols // 128) * 4), np.uint8)
    full[:, :s.shape[1]] = s
    return codes.astype(np.uint8), full.reshape(rows, -1, 4).transpose(1, 0, 2).copy()


def pack(codes, fmt):
    """The bytes that hold the codes."""
    return codes if fmt == "e4m3" else (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(held, fmt):
    if fmt == "e4m3":
        return held
    out = np.empty((held.shape[0], 2 * held.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = held & 15, held >> 4
    return out


def values(codes, scales, fmt):
    """float64 [rows, cols] of codes (one to an element) and scales."""
    rows, cols = codes.shape
    s = scales.transpose(1, 0, 2).reshape(rows, -1)[:, :cols // BLOCK].astype(np.float64)
    x = np.where(s == 255, np.nan, np.exp2(s - 127))
    table = np.append(TABLE[fmt], np.nan) if fmt == "e4m3" else TABLE[fmt]
    mag = table[codes & (SIGN[fmt] - 1)]
    return np.where(codes & SIGN[fmt], -mag, mag) * np.repeat(x, BLOCK, 1)


def rmsnorm(s, weight, eps):
    s = np.asarray(s, np.float64)
    return s * np.asarray(weight, np.float64) * (1.0 / np.sqrt((s * s).mean(-1, keepdims=True) + eps))


def silu_mul(g, u):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u
