"""Sampling from given uniform numbers, from its definition: sorted, in extended precision."""
from __future__ import annotations

import numpy as np


def sample_row(x, u, T=1.0, k=0, p=1.0, m=0.0) -> int:
    """The id of one row of logits (top-k, top-p, min-p in that order; T <= 0: greedy)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1
    if not T > 0:
        return int(np.argmax(x))
    if top == np.inf:
        x = np.where(x == np.inf, 0.0, -np.inf)
        top = 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = (x - top) / np.float64(T)
    w = np.where(x == -np.inf, 0.0, np.exp(np.where(np.isnan(z), 0.0, z).astype(np.longdouble)))
    w = np.where(w < 2.0 ** -45, 0.0, w).astype(np.longdouble)
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        before = np.concatenate([[np.longdouble(0)], c[:-1]])
        keep = before < np.longdouble(max(np.float64(p), 0.0)) * c[-1]
        keep[0] = True
        order = order[keep]
    order = np.sort(order[w[order] >= min(np.float64(m), 1.0)])
    order = order[w[order] > 0]
    c = np.cumsum(w[order])
    u = min(max(np.float64(u), 0.0), 1.0) if u == u else 0.0
    return int(order[min(int(np.searchsorted(c, np.longdouble(u) * c[-1], side="right")), len(order) - 1)])
