"""A KV cache in pages in float64: where a token lies, the values that pages hold, rotary positions, and the attention of new
tokens over one sequence. Pages are [pages, kv heads, page size, d] of bf16 values or e4m3 codes with scale bytes
[.., d / 32] (``oracle/mx.py``); token t of a cache row is row t % size of page table[row, t // size].
"""
from __future__ import annotations

import numpy as np

from . import mx


def quantize(x):
    """(codes, scales) of rows [..., d]: e4m3 codes and one scale byte per 32 elements."""
    x = np.asarray(x, np.float64)
    codes, scales = mx.quantize(x.reshape(-1, x.shape[-1]), "e4m3")
    s = scales.transpose(1, 0, 2).reshape(codes.shape[0], -1)[:, :x.shape[-1] // mx.BLOCK]
    return codes.reshape(x.shape), s.reshape(*x.shape[:-1], -1)


def values(codes, scales):
    """float64 values of e4m3 pages."""
    table = np.append(mx.TABLE["e4m3"], np.nan)
    s = scales.astype(np.float64)
    f = np.where(s == 255, np.nan, np.exp2(s - 127)).repeat(mx.BLOCK, -1)
    return np.where(codes & 128, -1.0, 1.0) * table[codes & 127] * f


def page_of(table_row, token, size, pages):
    """The page of a token, None where there is none."""
    if not 0 <= token < len(table_row) * size or not 0 <= table_row[token // size] < pages:
        return None
    return int(table_row[token // size])


def rows_at(held, table_row, tokens):
    """held [pages, heads, size, d] at the given tokens: [heads, tokens, d], 0 without a page, and which have one."""
    pages, heads, size, d = held.shape
    out, there = np.zeros((heads, len(tokens), d), held.dtype), np.zeros(len(tokens), bool)
    for i, t in enumerate(tokens):
        p = page_of(table_row, int(t), size, pages)
        if p is not None:
            out[:, i], there[i] = held[p, :, t % size], True
    return out, there


def rotate(x, positions, inv_freq):
    """Rows x [tokens, heads, d] turned by their positions: pairs (i, i + d / 2)."""
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    h = x.shape[-1] // 2
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def visible(n, committed, fresh, anc):
    """Which of committed + fresh tokens node n sees."""
    new = np.arange(fresh)
    own = new <= n if anc is None else np.array([(int(anc[n]) >> m) & 1 for m in range(fresh)], bool)
    return np.concatenate([np.ones(committed, bool), own.reshape(-1)])


def attention(q, k, v, there, committed, fresh, anc, scale):
    """Node rows q [N, q heads, d] over k, v [kv heads, committed + fresh, d] (``there``: the tokens that have a page):
    (out, bound) for the first ``fresh`` nodes. ``bound`` is how far an fp32 computation with bf16 weights may be from out, before
    its own rounding: a weight p is off by 2^-8 of it (its bf16 rounding; the sum is that of the rounded weights) and by
    the error of its exponent, d + 8 roundings of 2^-24 of the sum of magnitudes of a score, at most e in any; sums over the tokens
    add a rounding each. So |sum w v - out| <= (2^-8 + 2 e + (tokens + 8) 2^-23) (sum w |v| + |out|)."""
    heads, d = q.shape[1], q.shape[2]
    group = heads // k.shape[0]
    out, bound = np.zeros((fresh, heads, d)), np.zeros((fresh, heads, d))
    for n in range(fresh):
        sees = visible(n, committed, fresh, anc) & there
        if not sees.any():
            continue
        for h in range(heads):
            kk, vv = k[h // group][sees], v[h // group][sees]
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ q[n, h] * scale
                e = (d + 8) * 2.0 ** -24 * abs(scale) * (np.abs(kk) @ np.abs(q[n, h])).max() + 2.0 ** -22 * (1 + np.abs(s).max())
                w = np.exp(s - s.max())
                w /= w.sum()
                out[n, h] = w @ vv
                bound[n, h] = (2.0 ** -8 + 2 * e + (len(s) + 8) * 2.0 ** -23) * (w @ np.abs(vv) + np.abs(out[n, h]))
    return out, bound
