"""Heads normalized and rotated, E2M1 codes under E8M0 scales, and attention over them, in 64 bits (CPU oracle, test
infrastructure only)."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def rotate(x, table, positions, first, dims, style, inverse=False):
    """float64 x [T, heads, width] with its dims turned; table [P, dims] cosines then sines."""
    x = np.array(x, np.float64)
    if not dims:
        return x
    row = np.asarray(table, np.float64)[positions][:, None]
    c, s = row[..., :dims // 2], row[..., dims // 2:] * (-1 if inverse else 1)
    i = np.arange(dims // 2)
    a, b = (first + i, first + i + dims // 2) if style == "halves" else (first + 2 * i, first + 2 * i + 1)
    p, q = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = p * c - q * s, q * c + p * s
    return x


def heads(x, table=None, positions=None, *, norm=0, weight=None, first=0, dims=0, style="pairs", eps=1e-6, inverse=False):
    x = np.array(x, np.float64)
    if norm:
        root = np.sqrt(np.mean(x[..., :norm] ** 2, -1, keepdims=True) + eps)
        x[..., :norm] = x[..., :norm] / root * (1 if weight is None else np.asarray(weight, np.float64))
    return rotate(x, table, positions, first, dims, style, inverse)


def heads_backward(dy, x, table=None, positions=None, *, norm=0, weight=None, first=0, dims=0, style="pairs", eps=1e-6,
                   inverse=False):
    """(dx, dweight) for y = heads(x): from dy turned back, by the quotient rule."""
    g = rotate(dy, table, positions, first, dims, style, not inverse)
    if not norm:
        return g, None
    xn, gn = np.asarray(x, np.float64)[..., :norm], g[..., :norm]
    w = np.ones(norm) if weight is None else np.asarray(weight, np.float64)
    square = np.mean(xn ** 2, -1, keepdims=True) + eps
    dweight = np.sum(gn * xn / np.sqrt(square), (0, 1))
    dn = w * gn / np.sqrt(square) - xn * np.sum(w * gn * xn, -1, keepdims=True) / (norm * square ** 1.5)
    return np.concatenate([dn, g[..., norm:]], -1), dweight


def encode(x):
    """(codes [..., width] 0-15, scale bytes [..., width / 32]) of values that BF16 holds: the smallest power of two, at
    most 2^125, that keeps the block's largest magnitude (at least 1e-4) within 6; nearest code, ties to the even one; an
    infinity or NaN gives scale 255 and codes 0."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(blocks).all(-1)
    amax = np.where(finite, np.maximum(np.abs(np.where(np.isfinite(blocks), blocks, 0)).max(-1), np.float32(1e-4)), 1.0)
    m, k = np.frexp(amax / 6)                       # amax / 6 = m 2^k, m in [0.5, 1): the power at or above it
    e = np.minimum(np.where(m == 0.5, k - 1, k), 125)
    y = np.where(finite[..., None], np.abs(blocks), 0) / np.exp2(e)[..., None]
    distance = np.abs(y[..., None] - GRID)
    near = distance.min(-1, keepdims=True)
    code = np.argmax((distance == near) * (1 + (np.arange(8) % 2 == 0)), -1)   # an even code before an odd one
    code = np.where(finite[..., None], code + 8 * np.signbit(blocks), 0).astype(np.uint8)
    return code.reshape(x.shape), np.where(finite, e + 127, 255).astype(np.uint8)


def decode(codes, scales):
    """float64 values of codes 0-15 [..., width] and scale bytes [..., width / 32]."""
    codes = np.asarray(codes)
    v = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(np.asarray(scales) == 255, np.nan, np.exp2(np.asarray(scales, np.float64) - 127))
    return (v.reshape(*v.shape[:-1], -1, 32) * s[..., None]).reshape(codes.shape)


def pack(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def attend(q, keys, values, lengths, counts, scale, window=0, sinks=None, hidden=None):
    """(out [T, heads, value width], lse [T, heads], magnitude [T, heads, value width]) for q [T, heads, width] and keys,
    values [B][length][key heads][...]: a sequence's rows are its last counts[b] positions. hidden [B][length]: tokens
    that nobody sees. A NaN in a token's keys or values makes its whole row NaN for those who see it.

    magnitude: sum of p |v| / total, what the rounding of each probability is relative to."""
    t, h = q.shape[:2]
    out, lse, size = (np.zeros((t, h, v)) for v in (values[0].shape[-1] if len(values) else 1, 1, values[0].shape[-1] if len(values) else 1))
    lse = np.full((t, h), -np.inf)
    row = 0
    for b, n in enumerate(counts):
        k, v = np.asarray(keys[b], np.float64), np.asarray(values[b], np.float64)
        length = int(lengths[b])
        group = h // k.shape[1]
        bad = np.isnan(k).any(-1) | np.isnan(v).any(-1)
        for i in range(n):
            at = length - n + i
            seen = np.arange(length) <= at
            if window:
                seen &= np.arange(length) > at - window
            if hidden is not None:
                seen &= ~hidden[b][:length]
            tokens = np.flatnonzero(seen)
            for j in range(h):
                if tokens.size:
                    if bad[tokens, j // group].any():
                        out[row, j], lse[row, j], size[row, j] = np.nan, np.nan, np.nan
                        continue
                    s = k[tokens, j // group] @ q[row, j].astype(np.float64) * scale
                    top = s.max()
                    p = np.exp(s - top)
                    lse[row, j] = np.log(p.sum()) + top
                    total = p.sum() + (0 if sinks is None else np.exp(float(sinks[j]) - top))
                    out[row, j] = p @ v[tokens, j // group] / total
                    size[row, j] = p @ np.abs(v[tokens, j // group]) / total
            row += 1
    return out, lse, size
