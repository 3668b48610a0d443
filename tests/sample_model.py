"""The choice of a token in 64 bits on the host, from the definition, for the tests."""
from __future__ import annotations

import numpy as np


def keep(x, temperature, top_k, top_p, min_p):
    """(ids in index order, their weights, how near the nearest border of top_p or min_p is, relative to the whole)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    on = np.flatnonzero(x > -np.inf)
    if on.size == 0:
        return on, np.zeros(0), np.inf
    ids = on[np.argsort(-x[on], kind="stable")]
    m = x[ids[0]]
    if not temperature > 0:
        return ids[:1], np.ones(1), np.inf
    f = lambda v: float(np.float32(v))
    with np.errstate(all="ignore"):
        d = np.where(x[ids] == m, 0.0, x[ids] - m)
        w = np.where(d == -np.inf, 0.0, np.exp(d / f(temperature)))
    near = np.inf
    if top_k > 0:
        ids, w = ids[:top_k], w[:top_k]
    if top_p <= 0:
        ids, w = ids[:1], w[:1]
    elif top_p < 1:
        run, want = np.cumsum(w), f(top_p) * w.sum()
        n = int(np.searchsorted(run, want, side="left")) + 1
        near = np.min(np.abs(run - want)) / w.sum()
        ids, w = ids[:n], w[:n]
    if min_p > 0:
        least = min(f(min_p), 1.0)
        near = min([near] + np.abs(w[w < 1] - least).tolist())  # (the largest weigh 1 exactly)
        on = w >= least
        ids, w = ids[on], w[on]
    by = np.argsort(ids)
    return ids[by], w[by], near


def choose(x, u, temperature, top_k, top_p, min_p):
    """(token, probability, how near the nearest border is)."""
    ids, w, near = keep(x, temperature, top_k, top_p, min_p)
    if ids.size == 0:
        return -1, 0.0, near
    run = np.cumsum(w)
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    if u > 0:
        near = min(near, np.min(np.abs(run[:-1] - u * run[-1])) / run[-1] if len(run) > 1 else np.inf)
    if at >= len(ids):
        at = int(np.flatnonzero(w > 0)[-1])
    return int(ids[at]), w[at] / run[-1], near


def slack(x, temperature):
    """How near a border may be and the choice differ: every weight is rounded to a whole 2^-U of the largest (half of one
    each), and computed to 2^-45 of itself."""
    vocab = len(x)
    bits = 1
    while (1 << bits) <= vocab:
        bits += 1
    return vocab * 2.0 ** -(min(51, 62 - bits) + 1) + 2.0**-44
