"""Tokens sorted by expert and back, in 64 bits (CPU oracle, test infrastructure only).

Restates the device operators from their definitions: the pairs of a [T, k] routing table ordered by expert, then by
pair index (participation's expert-major, ascending-token order, src/vesper/moe.py:18-30); a token's result is the
weighted sum of its rows, the shared row last (MoEAccumulator, src/vesper/moe.py:42-148). Sums are float64, so a test
knows both the value and the sum of magnitudes that bounds an FP32 evaluation's error.
"""

from __future__ import annotations

import numpy as np


def plan(ids, experts: int):
    """(first [experts + 1], pair_row [T, k], row_pair [T k]) by visiting the experts in turn."""
    ids = np.asarray(ids)
    flat = ids.reshape(-1)
    pair_row = np.full(flat.size, -1, np.int32)
    order, first = [], [0]
    for e in range(experts):
        own = np.flatnonzero(flat == e)
        pair_row[own] = first[-1] + np.arange(own.size)
        order.extend(own.tolist())
        first.append(first[-1] + own.size)
    order.extend(np.flatnonzero((flat < 0) | (flat >= experts)).tolist())
    return np.asarray(first, np.int32), pair_row.reshape(ids.shape), np.asarray(order, np.int32)


def combine(rows, pair_row, weights=None, shared=None):
    """(y, magnitude) [T, width] float64: the sums and the sums of the terms' magnitudes."""
    t, k = pair_row.shape
    y = np.zeros((t, rows.shape[1]))
    size = np.zeros_like(y)
    for token in range(t):
        for j in range(k):
            if pair_row[token, j] >= 0:
                term = rows[pair_row[token, j]].astype(np.float64) * (1.0 if weights is None else
                                                                      np.float64(weights[token, j]))
                y[token] += term
                size[token] += np.abs(term)
    if shared is not None:
        y += shared.astype(np.float64)
        size += np.abs(shared.astype(np.float64))
    return y, size


def combine_backward(dy, rows, pair_row, weights=None):
    """(drows [T k, width], dweights [T, k], magnitude of the dot products [T, k]) float64; rows without a pair zero."""
    t, k = pair_row.shape
    drows = np.zeros((t * k, dy.shape[1]))
    dweights, size = np.zeros((t, k)), np.zeros((t, k))
    for token in range(t):
        g = dy[token].astype(np.float64)
        for j in range(k):
            r = pair_row[token, j]
            if r >= 0:
                drows[r] = g * (1.0 if weights is None else np.float64(weights[token, j]))
                terms = rows[r].astype(np.float64) * g
                dweights[token, j], size[token, j] = terms.sum(), np.abs(terms).sum()
    return drows, dweights, size
