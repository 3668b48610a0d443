"""Turned keys that keep and retain have closed up, on the GPU: the tokens behind them are turned by the positions that they have
in the text, and attention sees the distances that it saw before."""
from __future__ import annotations

import numpy as np
import pytest

from barracuda_amd import KvCache, Rotary
from tests.kv_model import attend, visible
from tests.rotary_model import depths, turned
from tests.test_gpu_kv_cache import _t
from tests.test_gpu_paged import compare, tolerance

pytestmark = pytest.mark.gpu


class _Model:
    """Every sequence's keys, values and positions, and each step against 64 bits."""

    def __init__(self, dev, rng, h, hkv, d, page, layers, **rotary):
        self.dev, self.rng, self.h, self.hkv, self.d = dev, rng, h, hkv, d
        self.cache, self.rotary = KvCache(layers, 96, page, hkv, d, dev), Rotary(d, device=dev, **rotary)
        self.held = {}

    def sequence(self):
        s = self.cache.new_sequence()
        self.held[s] = [([], [], []) for _ in range(self.cache.layers)]
        return s

    def step(self, items, parents=None):
        r, total = self.rotary, sum(n for _, n in items)
        step = self.cache.batch(items, parents)
        turn = lambda x, at: turned(x, np.asarray(at)[:, None], r.freqs, r.dim, r.interleaved, r.scale)
        for layer in range(self.cache.layers):
            q, k, v = (self.rng.standard_normal((total, n, self.d), dtype=np.float32) for n in (self.h, self.hkv, self.hkv))
            tk = _t(k, self.dev)
            out = self.cache.append_rotary(step, layer, r, _t(q, self.dev), tk, _t(v, self.dev))
            y, tq = self.cache.attention(step, layer, out).to_numpy(), out.to_numpy()
            assert np.array_equal(tk.to_numpy(), k)
            pool = self.cache.k.to_numpy()[layer]
            for i, (s, n) in enumerate(items):
                if n == 0:
                    continue
                rows = slice(int(step.start[i]), int(step.start[i + 1]))
                keys, values, where = self.held[s][layer]
                first = len(keys)
                at = (where[-1] + 1 if where else 0) + np.array(depths(parents[i]) if parents else range(n))
                want, tol = turn(q[rows], at)
                assert np.all(np.abs(tq[rows] - want) <= tol)
                want, tol = turn(k[rows], at)
                pages = self.cache.pages(s)
                got = np.stack([pool[pages[j // self.cache.page_size], :, j % self.cache.page_size] for j in range(first, first + n)])
                assert np.all(np.abs(got - want) <= tol)
                keys.extend(want.astype(np.float32))
                values.extend(v[rows])
                where.extend(at.tolist())
                scale = float(np.float32(1.0) / np.sqrt(np.float32(self.d)))
                ks, vs = np.stack(keys), np.stack(values)
                want = attend(tq[rows], ks, vs, visible(first, n, 0, 0, parents[i] if parents else None), scale)
                # a key's columns are off by 5 * 2^-24 of a pair's two magnitudes, which sum to at most sqrt(2) of their length: a
                # score by that of the lengths' product, a weighted mean by twice as much (numerator and denominator)
                s_max = scale * np.sqrt((tq[rows].astype(np.float64) ** 2).sum(-1).max() * (ks.astype(np.float64) ** 2).sum(-1).max())
                compare(y[rows], want, tolerance(tq[rows], ks, vs, scale, len(keys))
                        + 2 * 2 * 5 * 2.0**-24 * r.scale * s_max * np.abs(vs).max())
        return step

    def _only(self, s, ids):
        for lists in self.held[s]:
            for x in lists:
                x[:] = [x[j] for j in ids]

    def retain(self, s, ids):
        self.cache.retain(s, ids)
        self._only(s, ids)

    def keep(self, step, kept):
        self.cache.keep(step, kept)
        for s, n, ids in zip(step.sequences, step.counts, kept):
            old = len(self.held[s][0][0]) - n
            self._only(s, list(range(old)) + [old + x for x in ids])


@pytest.mark.parametrize("h,hkv,d,page,rotary", [(4, 2, 64, 16, {}), (3, 3, 80, 5, {"dim": 40, "interleaved": True, "base": 500.0}),
                                                 (8, 1, 128, 8, {"scaling": "linear", "factor": 4.0}), (2, 1, 33, 3, {"dim": 20})])
def test_sinks_and_the_newest_keys(dev, h, hkv, d, page, rotary):
    """The beginning and the newest keys stay, twice; tokens, a chunk and drafts follow, beside a sequence that keeps all."""
    m = _Model(dev, np.random.default_rng(d), h, hkv, d, page, 2, **rotary)
    a, b = m.sequence(), m.sequence()
    m.step([(a, 90), (b, 17)])
    m.retain(a, list(range(4)) + list(range(61, 90)))
    m.step([(a, 1), (b, 1)])
    m.step([(b, 0), (a, 9)])
    m.retain(a, list(range(4)) + list(range(20, 43)))
    step = m.step([(a, 5), (b, 3)], parents=[[-1, 0, 0, 2, -1], [-1, 0, 1]])
    m.keep(step, [[0, 2, 3], [0, 2]])  # a branch; and a list with a gap
    m.step([(a, 1), (b, 1)])
    c = m.cache.fork(a)
    m.held[c] = [tuple(list(x) for x in lists) for lists in m.held[a]]
    m.cache.truncate(a, 3)
    m._only(a, range(3))
    m.step([(a, 2), (c, 1), (b, 1)])


def test_the_fastest_pair_at_the_furthest_positions(dev):
    """Angles of up to 2^50: cosines and sines are still those of the product in 64 bits."""
    x = np.random.default_rng(1).standard_normal((1, 2, 64, 4), dtype=np.float32)
    r = Rotary(4, freqs=[2.0**19, 523456.789], device=dev)
    for first in (2**31 - 64, -(2**31) + 1, 12345678):
        y, tol = turned(x, first + np.arange(64), r.freqs, 4, False, 1.0)
        assert np.all(np.abs(_t(x, dev).rotary(r, first=first).to_numpy() - y) <= tol)
