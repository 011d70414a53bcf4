"""The operators on given logits in plain 64-bit numpy, straight from their definitions."""
import math

import numpy as np


def top_reference(logits, k, T):
    """(indices (n, k), lse (n,)) for float64 logits (n, V): value descending (NaN first), index ascending."""
    n, V = logits.shape
    indices = np.empty((n, k), dtype=np.int64)
    lse = np.empty(n)
    for r in range(n):
        row = logits[r]
        order = np.lexsort((np.arange(V), -np.where(np.isnan(row), 0.0, row), ~np.isnan(row)))
        indices[r] = order[:k]
        if np.isnan(row).any():
            lse[r] = np.nan
            continue
        m = row.max()
        lse[r] = m if np.isinf(m) else m / T + math.log(np.exp((row - m) / T).sum())
    return indices, lse


def sample_reference(row, u, T, top_k, top_p, min_p):
    """(token, logprob) of one float64 row."""
    allowed = np.flatnonzero(row > -np.inf)  # not -inf, not NaN
    if len(allowed) == 0:
        return -1, -math.inf
    order = allowed[np.lexsort((allowed, -row[allowed]))]
    if T <= 0:
        return int(order[0]), 0.0
    if top_k > 0:
        order = order[:top_k]
    top = row[order[0]]
    d = np.where(row[order] == top, 0.0, -np.inf) if np.isinf(top) else (row[order] - top) / T
    w = np.exp(d)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        stay = before < top_p * w.sum()
        stay[0] = True
        order, d, w = order[stay], d[stay], w[stay]
    if min_p > 0:
        stay = w >= min(min_p, 1.0)
        order, d, w = order[stay], d[stay], w[stay]
    by_index = np.argsort(order)
    order, d, w = order[by_index], d[by_index], w[by_index]
    mass = np.cumsum(w)
    at = min(int(np.searchsorted(mass, min(max(u, 0.0), 1.0) * mass[-1], side="right")), len(w) - 1)
    while w[at] == 0.0:  # rounding of the last sums only
        at -= 1
    return int(order[at]), float(d[at] - math.log(mass[-1]))
