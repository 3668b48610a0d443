"""Batches as a serving program pads them: room for more rows and longer chunks than there are, sequences without
keys or tokens behind the real ones, a longest length that is not the longest."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Tensor
from barracuda_amd import _native as N
from barracuda_amd.kv_cache import _I32
from tests.test_gpu_paged import Case, _tree, compare, tolerance

pytestmark = pytest.mark.gpu

BATCHES = [([300, 1, 800], [1, 1, 1]), ([300, 90, 700], [40, 3, 100]), ([2500, 1900], [9, 30]), ([600, 500], [500, 17])]


def pad(c, more, rows, max_new, max_len):
    """`more` empty sequences behind c's, room for `rows` more rows; the tail of each array holds what must not be used."""
    b = len(c.lens)
    start = np.concatenate([c.start, np.full(more, c.start[-1])])
    lens = np.concatenate([c.lens, np.arange(more) * 7])
    table = np.full((b + more, c.pool.table.shape[1]), 2**30, np.int32)
    table[:b] = c.pool.table
    parents = [] if c.parents is None else [x for t in c.parents for x in t] + [5] * rows
    c.i32 = _I32(c.dev, start, lens, table, parents)
    c.kv.table = c.i32.ptrs[2]
    c.batch = N.KvBatch(b + more, c.total + rows, max_new, max_len, c.i32.ptrs[0], c.i32.ptrs[1])


@pytest.mark.parametrize("d", [3, 6, 64, 128, 200, 300])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_padded_batches(dev, d, tree):
    rng = np.random.default_rng(d)
    for lens, news in BATCHES:
        if tree:
            news = [min(n, 128) for n in news]
        parents = [_tree(rng, n, True) for n in news] if tree else None
        c = Case(dev, lens, news, 4, 2, d, 16, 200, 3, parents=parents, tail_rows=75)
        tol = tolerance(c.q, c.pool.k, c.pool.v, c.scale, max(lens))
        want = c.want()
        for more, rows, max_new, max_len in ((0, 75, 128, 4000), (70, 0, max(news), 0), (3, 75, 100, 2**31 - 1), (200, 60, 128, 10)):
            max_new = max(max_new, max(news))
            print(f"padded d={d} tree={tree} lens={lens} more={more} rows={rows} max_new={max_new} max_len={max_len}", flush=True)
            pad(c, more, rows, max_new, max_len)
            dev.upload(c.po - 4 * c.misalign, np.full(c.to.len(), 7.0, np.float32))
            dev.check(c.call(dev._lib, dev.ctx), "attention")
            compare(c.output(), want, tol)


@pytest.mark.parametrize("d", [5, 64])
def test_append_of_padded_batches(dev, d):
    for lens, news in BATCHES:
        c = Case(dev, lens, news, 2, 2, d, 16)
        rng = np.random.default_rng(d)
        new = rng.standard_normal((2, c.total + 50, 2, d), dtype=np.float32)
        want = [x.copy() for x in (c.pool.k, c.pool.v)]
        for b, (length, n) in enumerate(zip(lens, news)):
            j = np.arange(length - n, length)
            for x, y in zip(want, new):
                x[c.pool.table[b, j // 16], :, j % 16] = y[c.start[b]:c.start[b + 1]]
        t = [Tensor.from_data(x, list(x.shape), dev) for x in new]
        row = N.AttnLayout(0, d, 2 * d)
        for more, rows, max_new in ((0, 50, 600), (90, 31, max(news)), (5, 0, 2**31 - 1)):
            c.upload()
            pad(c, more, rows, max_new, 0)
            dev.check(dev._lib.bch_kv_append(dev.ctx, c.kv, c.batch, C.c_void_p(t[0].ptr), row, C.c_void_p(t[1].ptr), row),
                      "append")
            for pool, x in zip((c.tk, c.tv), want):
                assert np.array_equal(pool.to_numpy().reshape(x.shape), x), (more, rows, max_new)
