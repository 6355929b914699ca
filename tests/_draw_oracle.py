"""Draws from truncated log-weights in numpy, entry by entry from the definition (test infrastructure)."""
import math

import numpy as np


def kept_entries(l, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(indices in index order, their weights, z of them) of one row of float64 log-weights."""
    alive = [i for i in range(len(l)) if l[i] > -math.inf]       # (false for NaN)
    if not alive:
        return np.zeros(0, dtype=np.int64), np.zeros(0), np.zeros(0)
    l = np.asarray(l, dtype=np.float64)
    alive = np.asarray(alive)
    order = alive[np.argsort(-l[alive], kind="stable")]
    best = l[order[0]]
    if not temperature > 0:
        return order[:1], np.ones(1), np.zeros(1)
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l[order] == best, 0.0, (l[order] - best) / temperature)
    w = np.exp(z)
    n = len(order)
    if top_k is not None and top_k > 0:
        n = min(n, int(top_k))
    if top_p is not None and top_p < 1.0:
        if top_p <= 0.0:
            n = 1
        else:
            c = np.cumsum(w[:n])
            n = min(n, 1 + int(np.searchsorted(c, top_p * c[-1], side="left")))
    if min_p is not None and min_p > 0:
        n = int(np.count_nonzero(w[:n] >= min(min_p, 1.0)))
    at = np.argsort(order[:n])
    return order[:n][at], w[:n][at], z[:n][at]


def draw_row(l, u, **settings):
    idx, w, z = kept_entries(l, **settings)
    out, logp = np.full(len(u), -1, dtype=np.int64), np.full(len(u), -math.inf)
    if len(idx) == 0:
        return out, logp
    c = np.cumsum(w)
    last = int(np.flatnonzero(w > 0)[-1])
    log_z = math.log(math.fsum(w.tolist()))                      # (a running sum of V terms would be off by up to V half steps itself)
    for s, x in enumerate(u):
        j = min(int(np.searchsorted(c, x * c[-1], side="right")), last)
        out[s], logp[s] = idx[j], z[j] - log_z
    return out, logp
