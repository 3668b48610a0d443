"""Plain forms of the paged cache and its attention, in 64 bits on the host, for the tests."""
from __future__ import annotations

import numpy as np


def visible(first, n, window, sinks, parents=None):
    """[n, first + n] of truth values: which keys each of n rows at the end of first + n keys sees.  first may
    be negative (more rows than keys); then only keys from 0 on are there."""
    length = first + n
    see = np.zeros((n, max(length, 0)), dtype=bool)
    if parents is None:
        pos = [first + i for i in range(n)]
        chains = [[(j, first + j) for j in range(i + 1)] for i in range(n)]
    else:
        depth, chains = [], []
        for i, p in enumerate(parents):
            ok = 0 <= p < i
            depth.append(depth[p] + 1 if ok else 0)
            chains.append((chains[p] if ok else []) + [(i, first + depth[i])])
        pos = [first + d for d in depth]
    for i in range(n):
        keys = [(j, j) for j in range(max(first, 0))] + [(first + a, at) for a, at in chains[i]]
        for j, at in keys:
            if j >= 0 and (window == 0 or pos[i] - at < window or at < sinks):
                see[i, j] = True
    return see


def attend(q, k, v, see, scale):
    """q [n, H, D], k and v [L, Hkv, D], see [n, L] -> [n, H, D] in float64; rows that see nothing, or nothing
    above -inf, are zeros.  Values that a row does not see do not reach it."""
    n, h, d = q.shape
    hkv = k.shape[1]
    out = np.zeros((n, h, d))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    with np.errstate(all="ignore"):
        for i in range(n):
            keys = np.flatnonzero(see[i])
            if keys.size == 0:
                continue
            for head in range(h):
                kv = head // (h // hkv)
                s = scale * (k[keys, kv] @ q[i, head])
                on = s != -np.inf
                if not on.any():
                    continue
                s, vv = s[on], v[keys[on], kv]
                m = s.max()
                p = np.exp(s - m)
                out[i, head] = (p[:, None] * vv).sum(0) / p.sum()
    return out


class Pages:
    """A pool of pages with sequences on scattered pages, as numpy arrays."""

    def __init__(self, rng, lens, hkv, d, page, spare=3, fill=None):
        held = [-(-n // page) for n in lens]
        self.num = sum(held) + spare
        order = rng.permutation(self.num).astype(np.int32)
        self.table = np.full((len(lens), max(1, max(held))), -1, np.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.num, hkv, page, d)
        if fill is None:
            self.k, self.v = (rng.standard_normal(shape, dtype=np.float32) for _ in range(2))
        else:
            self.k, self.v = (np.full(shape, fill, np.float32) for _ in range(2))
            for b, n in enumerate(lens):  # what is not a key stays as filled
                for j in range(n):
                    p, s = self.table[b, j // page], j % page
                    self.k[p, :, s] = rng.standard_normal((hkv, d), dtype=np.float32)
                    self.v[p, :, s] = rng.standard_normal((hkv, d), dtype=np.float32)
        self.page = page

    def keys(self, b, length, pool):
        """[length, Hkv, D] of sequence b, and which of them are held."""
        j = np.arange(length)
        p = self.table[b, j // self.page]
        on = (p >= 0) & (p < self.num)
        return pool[np.where(on, p, 0), :, j % self.page], on
