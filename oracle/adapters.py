"""Low-rank adapters beside a projection, in 64 bits (CPU oracle, test infrastructure only):
y[t] = base[t] + scale up (down x[t]) with the adapter of slot ids[t], base[t] where there is none.

`apply` also gives what bounds an FP32 evaluation: the magnitude of the terms of each result."""

from __future__ import annotations

import numpy as np


def apply(x, ids, base, adapters):
    """(y, magnitude) [T, rows] float64; adapters {slot: (down [rank, width], up [rows, rank], scale)} as values.

    magnitude = |base| + |scale| |up| (|down| |x|): the sum of all the products' magnitudes."""
    x, y = np.asarray(x, np.float64), np.asarray(base, np.float64).copy()
    size = np.abs(y)
    ids = np.asarray(ids)
    for slot, values in adapters.items():
        down, up, scale = (np.asarray(a, np.float64) for a in values)
        own = np.flatnonzero(ids == slot)
        y[own] += scale * (x[own] @ down.T @ up.T)
        size[own] += np.abs(scale) * (np.abs(x[own]) @ np.abs(down).T @ np.abs(up).T)
    return y, size
