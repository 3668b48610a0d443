"""Calls over so many sequences, with one long chunk among them, that a grid cannot have a workgroup for each place
that the longest chunk's length gives every sequence.  The single tokens share a few pages; a sample of the rows is
compared with plain forms in 64 bits, and every row has to be written."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Tensor
from barracuda_amd import _native as N
from barracuda_amd.kv_cache import _I32
from tests.kv_model import attend, visible
from tests.test_gpu_paged import compare, tolerance
from tests.test_paged_route import kernels

pytestmark = pytest.mark.gpu


class Crowd:
    """b sequences of a token each, but `at` with `new` of them behind `before` keys."""

    def __init__(self, dev, b, at, new, before, h, hkv, d, page=8, window=0, sinks=0, tree=None):
        rng = np.random.default_rng(b + d)
        self.dev, self.h, self.hkv, self.d, self.page = dev, h, hkv, d, page
        self.window, self.sinks, self.tree, self.at = window, sinks, tree, at
        news = np.ones(b, np.int64)
        news[at] = new
        self.start = np.concatenate([[0], np.cumsum(news)])
        self.total = int(self.start[-1])
        self.lens = rng.integers(1, 2 * page + 1, b).astype(np.int32)
        self.lens[at] = before + new
        held = -(-(before + new) // page)
        self.width, self.num = max(2, held), held + 50
        self.table = np.full((b, self.width), -1, np.int32)
        self.table[:, :2] = rng.integers(held, self.num, (b, 2))
        self.table[at, :held] = rng.permutation(held)
        self.k, self.v = (rng.standard_normal((self.num, hkv, page, d), dtype=np.float32) for _ in range(2))
        self.q = rng.standard_normal((self.total, h, d), dtype=np.float32)
        parents = []
        if tree is not None:
            parents = np.full(self.total, -1, np.int32)
            parents[self.start[at]:self.start[at + 1]] = tree
        self.tk, self.tv, self.tq = (Tensor.from_data(x, list(x.shape), dev) for x in (self.k, self.v, self.q))
        self.to = Tensor.from_data(np.full(self.q.shape, 7.0, np.float32), list(self.q.shape), dev)
        self.i32 = _I32(dev, self.start, self.lens, self.table, parents)
        lay = N.AttnLayout(hkv * page * d, page * d, d)
        self.kv = N.KvPages(self.tk.ptr, self.tv.ptr, lay, lay, self.num, page, hkv, d, self.i32.ptrs[2], self.width)
        self.batch = N.KvBatch(b, self.total, new, int(self.lens.max()), self.i32.ptrs[0], self.i32.ptrs[1])
        self.row = N.AttnLayout(0, d, h * d)

    def keys(self, s, pool):
        j = np.arange(self.lens[s])
        return pool[self.table[s, j // self.page], :, j % self.page]

    def check(self, some):
        dev = self.dev
        parent = C.c_void_p(self.i32.ptrs[3]) if self.tree is not None else None
        scale = float(1.0 / np.sqrt(self.d))
        dev.check(dev._lib.bch_sdpa_paged(dev.ctx, self.kv, self.batch, self.h, scale, self.window, self.sinks, parent,
                                          C.c_void_p(self.tq.ptr), self.row, C.c_void_p(self.to.ptr), self.row),
                  "attention")
        got = self.to.to_numpy().reshape(self.q.shape)
        assert not np.any(got[..., 0] == 7.0), "rows left as they were"
        rng = np.random.default_rng(1)
        b = self.batch.B
        for s in [0, self.at, b - 1] + list(rng.integers(0, b, some)):
            first, n = int(self.lens[s] - (self.start[s + 1] - self.start[s])), int(self.start[s + 1] - self.start[s])
            k, v = self.keys(s, self.k), self.keys(s, self.v)
            i = np.arange(n) if n <= 128 else np.unique(np.concatenate([[0, 1, n - 1], rng.integers(0, n, 60)]))
            if self.tree is not None:
                see = visible(first, n, self.window, self.sinks, list(self.tree) if s == self.at else [-1])
            else:
                back = (first + i)[:, None] - np.arange(len(k))[None, :]
                see = back >= 0
                if self.window:
                    see &= (back < self.window) | (np.arange(len(k)) < self.sinks)[None, :]
            rows = self.start[s] + i
            compare(got[rows], attend(self.q[rows], k, v, see, scale),
                    tolerance(self.q[rows], k, v, scale, len(k)))


@pytest.mark.parametrize("tree", [False, True])
def test_three_million_sequences(dev, tree):
    """Where once the short sequences' kernel did not run and their rows were left as they were."""
    b, new = 3000000, 16
    drafts = [-1, 0, 0, 1, 3, 2, 2, -1, 7, 8, 8, 5, 0, 12, 12, 9] if tree else None
    print(f"crowd b={b} tree={tree} {kernels(b, b + new - 1, new, 20, 4, 1, 8)}", flush=True)
    Crowd(dev, b, b // 3, new, 4, 4, 1, 8, tree=drafts).check(500)


@pytest.mark.parametrize("b,new,h,hkv,d,window,sinks", [(8192, 8192, 32, 4, 8, 64, 2), (8192, 8192, 32, 4, 131, 50, 0),
                                                        (16384, 1024, 8, 1, 5, 0, 0)])
def test_a_long_chunk_beside_many_sequences(dev, b, new, h, hkv, d, window, sinks):
    k = kernels(b, b + new - 1, new, new + 33, h, hkv, d, window, sinks)
    print(f"crowd b={b} new={new} h={h} hkv={hkv} d={d} {k}", flush=True)
    assert any(x is not True and x[1] < 0 for x in k.values()), "lists are not dealt out"
    Crowd(dev, b, b // 2, new, 33, h, hkv, d, page=16, window=window, sinks=sinks).check(200)


@pytest.mark.parametrize("d", [2, 300])
def test_a_chunk_beside_many_sequences_at_other_widths(dev, d):
    """Widths that take a workgroup a row and head: 2^24 and more of them by the longest chunk's length."""
    b, new, h, hkv = 1100, 8192, 2, 1
    print(f"crowd b={b} new={new} d={d} {kernels(b, b + new - 1, new, new + 5, h, hkv, d, 40, 1)}", flush=True)
    Crowd(dev, b, 700, new, 5, h, hkv, d, page=16, window=40, sinks=1).check(200)
    # and more rows that there are than one launch takes
    if d == 2:
        Crowd(dev, 1 << 22, 5, 7, 5, 4, 2, d, page=4).check(500)


def test_dense_batches_beyond_one_launch(dev):
    b, h, sq, d = 1 << 20, 3, 3, 2
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal((b, h, sq, d), dtype=np.float32) for _ in range(3))
    t = [Tensor.from_data(x, list(x.shape), dev) for x in (q, k, v)]
    got = t[0].sliding_window_attention(t[1], t[2], 2, 1).to_numpy().reshape(q.shape)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    see = visible(0, sq, 2, 1)
    for i in [0, b - 1] + list(rng.integers(0, b, 300)):
        want = attend(*(x[i].transpose(1, 0, 2) for x in (q, k, v)), see, scale)
        compare(got[i].transpose(1, 0, 2), want, tolerance(q[i], k[i], v[i], scale, sq))


@pytest.mark.parametrize("b,new,d", [(4096, 8193, 3), (4096, 8193, 4), (1 << 22, 9, 3), (1 << 22, 9, 4), (3, 1 << 25, 3)])
def test_append_of_batches_beyond_a_grid(dev, b, new, d):
    """2^24 and more places of two tokens by the longest chunk's length: every key into its page, bit for bit, and
    nothing beside them."""
    print(f"append b={b} new={new} d={d}", flush=True)
    rng = np.random.default_rng(b)
    page, at = 16, b // 2
    news = np.ones(b, np.int64)
    news[at] = new
    news[rng.integers(0, b, b // 5)] = 0
    news[[0, at]] = [1, new]
    start = np.concatenate([[0], np.cumsum(news)])
    total = int(start[-1])
    lens = np.minimum(news + rng.integers(0, 9, b), page)
    lens[at] = new + 21
    # every sequence has a page of its own, the long one as many as it needs
    held = -(-int(lens[at]) // page)
    table = np.full((b, held), -1, np.int32)
    table[:, 0] = rng.permutation(b)
    table[at] = [table[at, 0]] + list(range(b, b + held - 1))
    num = b + held
    new_k = rng.standard_normal((total, d), dtype=np.float32)
    new_v = new_k[::-1].copy()
    pool = [Tensor.from_data(np.full((num, page, d), 5.0, np.float32), [num, page, d], dev) for _ in range(2)]
    t = [Tensor.from_data(x, [total, d], dev) for x in (new_k, new_v)]
    i32 = _I32(dev, start, lens, table)
    lay, row = N.AttnLayout(page * d, page * d, d), N.AttnLayout(0, d, d)
    kv = N.KvPages(pool[0].ptr, pool[1].ptr, lay, lay, num, page, 1, d, i32.ptrs[2], held)
    batch = N.KvBatch(b, total, new, int(lens.max()), i32.ptrs[0], i32.ptrs[1])
    dev.check(dev._lib.bch_kv_append(dev.ctx, kv, batch, C.c_void_p(t[0].ptr), row, C.c_void_p(t[1].ptr), row), "append")
    which = np.repeat(np.arange(b), news)
    j = (lens - news - start[:-1])[which] + np.arange(total)
    p, slot = table[which, j // page], j % page
    for got, x in zip(pool, (new_k, new_v)):
        want = np.full((num, page, d), 5.0, np.float32)
        want[p, slot] = x
        assert np.array_equal(got.to_numpy().reshape(want.shape).view(np.uint32), want.view(np.uint32))
