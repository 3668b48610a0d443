"""Attention over a paged cache where the lists of keys stand in one line that is cut into equal shares, by the tile
kernels (D up to 128, and 129 to 256): workgroups that hold the end of one list, whole ones and the beginning of
another.  That a case is cut so, and what its workgroups hold, is worked out from the kernels' plan; results are
compared with plain forms in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from tests.kv_model import attend, visible
from tests.test_gpu_paged import Case, _tree, compare, tolerance
from tests.test_paged_route import kernels

pytestmark = pytest.mark.gpu

BLOCK = 32  # keys of a block of the tile kernels
OVER = {"tile": 4, "wide": 2}  # blocks that a list's beginning and end count as


def lists(lens, news, h, hkv, name, rows, window, sinks, tree):
    """Length in blocks of every list, in the line's order: the keys that any row of the sequence sees."""
    out = []
    for length, n in zip(lens, news):
        if n * (h // hkv) <= 48:  # the other kernel's
            continue
        first = length - n
        lo = max(0, first - window + 1) if window else 0
        s_hi = min(sinks, lo)
        m0 = lo // BLOCK
        ns = min(-(-s_hi // BLOCK), m0)
        blocks = ns + -(-length // BLOCK) - m0
        out += [blocks + OVER[name]] * (hkv * -(-n * (h // hkv) // rows))
    return out


def held(lengths, grid, least):
    """What each workgroup of an evenly cut line holds: (ends of lists, whole lists, beginnings)."""
    total = sum(lengths)
    share = max(least, -(-total // grid))
    # each list cut by itself: so much longer pieces that it is not done, with a margin
    assert len(lengths) >= grid or max(least, -(-total // (grid - len(lengths)))) > 1.08 * share, "lists cut one by one"
    out, at = [[0, 0, 0] for _ in range(grid)], 0
    for n in lengths:
        for w in range(at // share, (at + n - 1) // share + 1):
            a, e = max(at, w * share), min(at + n, (w + 1) * share)
            whole, begins = (a, e) == (at, at + n), a == at
            out[w][1 if whole else 2 if begins else 0] += 1
        at += n
    return out


class Line(Case):
    def seen(self, b):
        length, n = self.lens[b], self.news[b]
        first = length - n
        if self.parents is None:
            back = first + np.arange(n)[:, None] - np.arange(length)[None, :]
            see = back >= 0
            return see & ((back < self.window) | (np.arange(length) < self.sinks)) if self.window else see
        depth = []
        for i, p in enumerate(self.parents[b]):
            depth.append(depth[p] + 1 if 0 <= p < i else 0)
        back = first + np.array(depth)[:, None] - np.arange(first)[None, :]
        see = (back < self.window) | (np.arange(first) < self.sinks) if self.window else back >= 0
        # the drafts among themselves: their positions count from `first`
        sinks = max(0, self.sinks - first)
        return np.concatenate([see, visible(0, n, self.window, sinks, self.parents[b])], axis=1)

    def want(self):
        out = np.zeros((self.total, self.h, self.d))
        group = self.h // self.hkv
        for b, (length, n) in enumerate(zip(self.lens, self.news)):
            if n == 0:
                continue
            rows = slice(int(self.start[b]), int(self.start[b + 1]))
            (k, on), (v, _) = self.pool.keys(b, length, self.pool.k), self.pool.keys(b, length, self.pool.v)
            see = self.seen(b) & on
            if not (np.isfinite(k).all() and np.isfinite(v).all()):
                out[rows] = attend(self.q[rows], k, v, see, self.scale)
                continue
            k, v = k.astype(np.float64), v.astype(np.float64)
            for h in range(self.h):
                s = np.where(see, self.scale * (self.q[rows, h].astype(np.float64) @ k[:, h // group].T), -np.inf)
                p = np.exp(s - np.maximum(s.max(1, keepdims=True), -1e300))
                total = p.sum(1, keepdims=True)
                out[rows, h] = np.where(total > 0, (p @ v[:, h // group]) / np.where(total > 0, total, 1.0), 0.0)
        return out

    def workgroups(self):
        """The kernel, and what its workgroups hold; the case has to be one that is cut as a line."""
        k = kernels(len(self.lens), self.total, self.max_new, max(self.lens), self.h, self.hkv, self.d, self.window,
                    self.sinks)
        name = "tile" if self.d <= 128 else "wide"
        rows, shares, least = k[name]
        assert shares > 0 and k["combine"], k
        all_lists = lists(self.lens, self.news, self.h, self.hkv, name, rows, self.window, self.sinks, self.parents)
        return k, held(all_lists, shares, least)


def check_mixed(c):
    """Workgroups hold an end and a beginning, and, where lists differ enough in length, whole lists between them."""
    k, w = c.workgroups()
    some = sum(1 for x in w if all(x))
    print(f"line d={c.d} window={c.window} sequences={len(c.lens)} {k} mixed={some} used={sum(map(any, w))}", flush=True)
    assert sum(1 for x in w if x[0] and x[2]) >= 20 and (c.window or some >= 5)
    c.check()


def ragged(seed, b, longest, most):
    """Lengths and new tokens of b sequences: a few without any, with one, and short ones among longer ones."""
    rng = np.random.default_rng(seed)
    news = [int(x) for x in rng.integers(13, most + 1, b)]
    lens = [n + int(x) for n, x in zip(news, np.exp(rng.uniform(0, np.log(longest), b)))]
    lens[1], news[1] = longest + most, most
    lens[2], news[2] = 700, 0
    lens[3], news[3] = 900, 1
    lens[4], news[4] = 5, 20  # more rows than keys
    return lens, news


@pytest.mark.parametrize("d", [64, 100, 128, 192, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 40)])
def test_chunks(dev, d, window, sinks):
    lens, news = ragged(1, 40, 2200, 200) if d <= 128 else ragged(1, 28, 2200, 120)
    check_mixed(Line(dev, lens, news, 8, 2, d, 16, window, sinks))


@pytest.mark.parametrize("d", [64, 80, 128, 160, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 4)])
def test_trees_of_more_sequences_than_a_wavefront_looks_at(dev, d, window, sinks):
    rng = np.random.default_rng(d)
    h = 8 if d <= 128 else 4
    lens, news = ragged(2, 75, 1500, 60)
    lens[1], news[1] = 1500, 128
    lens[4], news[4] = 30, 25
    lens = [x + (400 if i % 5 else 0) for i, x in enumerate(lens)]
    parents = [_tree(rng, n, i % 2 == 0) for i, n in enumerate(news)]
    check_mixed(Line(dev, lens, news, h, 2, d, 16, window, sinks, parents=parents))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("d", [64, 128, 200])
def test_values_that_are_not_finite_in_every_piece(dev, d, bad):
    """Keys near the end of every sequence, which some of its rows see, hold `bad`, and so does all that is no key: a
    list is done again in whichever of a workgroup's pieces it is."""
    lens, news = ragged(3, 66, 1000, 34)
    lens = [x + 300 for x in lens]
    c = Line(dev, lens, news, 8, 2, d, 16, 900, 2, fill=bad)
    k, w = c.workgroups()
    assert sum(1 for x in w if sum(x) > 1) >= 20, "workgroups with several pieces"
    for b, (length, n) in enumerate(zip(lens, news)):
        if n > 1 and b % 4:
            j = length - 1 - n // 2
            p = c.pool.table[b, j // 16]
            c.pool.v[p, b % 2, j % 16, ::3] = bad
            c.pool.k[p, 1 - b % 2, j % 16, [1, d - 2]] = bad
    c.upload()
    c.check()


@pytest.mark.parametrize("d,h,hkv", [(64, 16, 2), (128, 16, 2), (256, 8, 2)])
def test_up_to_two_tiles_a_compute_unit_behind_long_histories(dev, d, h, hkv):
    """More full tiles than half the compute units, shared because the lists are long and much alike."""
    news = [600, 530, 610, 470] if d <= 128 else [580, 500, 560, 520]
    lens = [n + x for n, x in zip(news, (900, 1100, 700, 2000))]
    c = Line(dev, lens, news, h, hkv, d, 64)
    k, w = c.workgroups()
    name = "tile" if d <= 128 else "wide"
    full = c.total * h // k[name][0]
    print(f"line d={d} {k} full tiles {full}", flush=True)
    assert k[name][1] // 2 < full <= 2 * k[name][1]
    assert sum(1 for x in w if x[0] and x[2]) >= 20
    c.check()
