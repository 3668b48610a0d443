"""The paged cache's own calls (append, page copies, keep), bit for bit, and KvCache from prompt to eviction
with attention at every step, against the plain forms."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import KvCache, Tensor
from barracuda_amd import _native as N
from barracuda_amd.error import InvalidInput
from barracuda_amd.kv_cache import _I32
from tests.kv_model import Pages, attend, visible
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip
from tests.test_gpu_paged import compare, tolerance

pytestmark = pytest.mark.gpu


def _t(x, dev):
    return Tensor.from_data(x, list(x.shape), dev)


def _p(t):
    return C.c_void_p(t.ptr)


class Pool:
    """Layers of pools in HBM beside their numpy images."""

    def __init__(self, dev, rng, lens, hkv, d, page, layers=1, slots=False, pad=0, misalign=0):
        self.dev, self.hkv, self.d, self.page, self.layers = dev, hkv, d, page, layers
        self.slots, self.pad, self.misalign = slots, pad, misalign
        self.pages = [Pages(np.random.default_rng(7), lens, hkv, d, page) for _ in range(layers)]
        for p in self.pages:
            p.k, p.v = (rng.standard_normal(p.k.shape, dtype=np.float32) for _ in range(2))
        self.num, self.table = self.pages[0].num, self.pages[0].table
        w = d + pad
        self.layer = self.num * hkv * page * w
        self.tk, self.tv = (self._put([getattr(p, x) for p in self.pages]) for x in "kv")
        lay = (N.AttnLayout(hkv * page * w, w, hkv * w) if slots else N.AttnLayout(hkv * page * w, page * w, w))
        self.i32 = _I32(dev, self.table)
        self.kv = N.KvPages(self.tk.ptr + 4 * misalign, self.tv.ptr + 4 * misalign, lay, lay, self.num, page, hkv, d,
                            self.i32.ptrs[0], self.table.shape[1])

    def _put(self, xs):
        w = self.d + self.pad
        y = np.full((self.layers,) + xs[0].shape[:3] + (w,), 5.0, np.float32)
        for i, x in enumerate(xs):
            y[i, ..., :self.d] = x
        if self.slots:
            y = y.transpose(0, 1, 3, 2, 4)
        return Tensor.from_data(np.concatenate([np.zeros(self.misalign, np.float32), y.reshape(-1)]),
                                [y.size + self.misalign], self.dev)

    def check(self):
        """Every float of the pools, padding included, is the images'."""
        for t, x in ((self.tk, "k"), (self.tv, "v")):
            want = self._put([getattr(p, x) for p in self.pages]).to_numpy()
            assert np.array_equal(t.to_numpy(), want), x


SHAPES = [(1, 4, 3, 1, 0, 0, False), (2, 64, 16, 1, 0, 0, False), (8, 128, 16, 3, 0, 0, False), (3, 80, 24, 2, 4, 0, True),
          (2, 33, 5, 2, 0, 0, False), (4, 64, 8, 1, 0, 1, False), (4, 64, 8, 2, 3, 0, True), (5, 300, 7, 1, 0, 0, True)]


@pytest.mark.parametrize("hkv,d,page,layers,pad,misalign,slots", SHAPES)
@pytest.mark.parametrize("lens,news", [([1], [1]), ([40, 7, 33, 0], [1, 0, 33, 0]), ([100, 61], [59, 61]), ([3, 20], [5, 4])])
def test_append(dev, lens, news, hkv, d, page, layers, pad, misalign, slots):
    rng = np.random.default_rng(1)
    pool = Pool(dev, rng, lens, hkv, d, page, layers, slots, pad, misalign)
    start = np.concatenate([[0], np.cumsum(news)])
    total = int(start[-1])
    w = d + pad
    i32 = _I32(dev, start, lens)
    batch = N.KvBatch(len(lens), total, max(news), max(lens), *i32.ptrs)
    new = rng.standard_normal((2, total, hkv, w), dtype=np.float32)
    tn = [_t(np.concatenate([np.zeros(misalign, np.float32), x.reshape(-1)]), dev) for x in new]
    row = N.AttnLayout(0, w, hkv * w)
    args = [(C.c_void_p(t.ptr + 4 * misalign), row) for t in tn]
    dev.check(dev._lib.bch_kv_append(dev.ctx, pool.kv, batch, *args[0], *args[1]), "append")
    img = pool.pages[0]
    for b, (length, n) in enumerate(zip(lens, news)):
        for i in range(n):
            j = length - n + i
            if j >= 0:
                p = img.table[b, j // page]
                img.k[p, :, j % page], img.v[p, :, j % page] = new[0, start[b] + i, :, :d], new[1, start[b] + i, :, :d]
    pool.check()


def test_append_skips_pages_that_are_not_held(dev):
    rng = np.random.default_rng(2)
    pool = Pool(dev, rng, [20, 40], 2, 64, 8)
    pool.table[0, 2], pool.table[1, [1, 4]] = -1, [pool.num, 2**30]
    pool.i32 = _I32(dev, pool.table)
    pool.kv.table = pool.i32.ptrs[0]
    i32 = _I32(dev, [0, 20, 60], [20, 40])
    new = rng.standard_normal((2, 60, 2, 64), dtype=np.float32)
    row = N.AttnLayout(0, 64, 128)
    tk, tv = _t(new[0], dev), _t(new[1], dev)
    dev.check(dev._lib.bch_kv_append(dev.ctx, pool.kv, N.KvBatch(2, 60, 40, 40, *i32.ptrs), _p(tk), row, _p(tv), row), "append")
    img = pool.pages[0]
    for b, n, s0 in ((0, 20, 0), (1, 40, 20)):
        for j in range(n):
            p = pool.table[b, j // 8]
            if 0 <= p < pool.num:
                img.k[p, :, j % 8], img.v[p, :, j % 8] = new[0, s0 + j], new[1, s0 + j]
    pool.check()


@pytest.mark.parametrize("hkv,d,page,layers,pad,misalign,slots", SHAPES)
@pytest.mark.parametrize("n", [1, 3, 17])
def test_copy_pages(dev, hkv, d, page, layers, pad, misalign, slots, n):
    rng = np.random.default_rng(3)
    pool = Pool(dev, rng, [page * 2 * n], hkv, d, page, layers, slots, pad, misalign)
    order = rng.permutation(pool.num)
    src, dst = order[:n], order[n:2 * n]
    src = np.where(rng.random(n) < 0.3, src[0], src)  # one page to several
    arr = C.c_int * n
    dev.check(dev._lib.bch_kv_copy_pages(dev.ctx, pool.kv, layers, pool.layer, pool.layer, n, arr(*src), arr(*dst)), "copy")
    for img in pool.pages:
        img.k[dst], img.v[dst] = img.k[src], img.v[src]
    pool.check()


def test_copy_more_pages_than_one_launch_takes(dev):
    rng = np.random.default_rng(4)
    n = 1201
    pool = Pool(dev, rng, [2 * n], 1, 8, 1, 2)
    order = rng.permutation(pool.num)
    src, dst = order[:n], order[n:2 * n]
    arr = C.c_int * n
    dev.check(dev._lib.bch_kv_copy_pages(dev.ctx, pool.kv, 2, pool.layer, pool.layer, n, arr(*src), arr(*dst)), "copy")
    for img in pool.pages:
        img.k[dst], img.v[dst] = img.k[src], img.v[src]
    pool.check()


def _keep(pool, keep, to):
    start = np.concatenate([[0], np.cumsum([len(x) for x in keep])])
    flat = [x for k in keep for x in k]
    i32 = _I32(pool.dev, start, flat, to)
    pool.dev.check(pool.dev._lib.bch_kv_keep(pool.dev.ctx, pool.kv, pool.layers, pool.layer, pool.layer, len(keep),
                                             len(flat), *[C.c_void_p(p) for p in i32.ptrs]), "keep")
    for img in pool.pages:
        for b, ids in enumerate(keep):
            for i, j in enumerate(ids):
                t = to[b] + i
                a, c = img.table[b, j // pool.page], img.table[b, t // pool.page]
                img.k[c, :, t % pool.page], img.v[c, :, t % pool.page] = (img.k[a, :, j % pool.page].copy(),
                                                                         img.v[a, :, j % pool.page].copy())


@pytest.mark.parametrize("hkv,d,page,layers,pad,misalign,slots", SHAPES)
def test_keep(dev, hkv, d, page, layers, pad, misalign, slots):
    rng = np.random.default_rng(5)
    lens = [90, 50, 300, 64]
    pool = Pool(dev, rng, lens, hkv, d, page, layers, slots, pad, misalign)
    drafts = sorted(rng.choice(20, 7, replace=False) + 70)
    _keep(pool, [drafts, [], sorted(rng.choice(300, 170, replace=False)), list(range(64))], [70, 3, 0, 0])
    pool.check()


def test_keep_of_keys_one_up_and_far_apart(dev):
    """Every key one place down (each is read before the next takes its place), and ranges that do not meet."""
    rng = np.random.default_rng(6)
    pool = Pool(dev, rng, [1000, 900], 4, 128, 16, 2)
    _keep(pool, [list(range(1, 1000)), list(range(500, 900))], [0, 4])
    pool.check()


def test_captured_append_and_keep(dev):
    """Append, keep and a page copy in one graph, replayed with other lengths."""
    hip = _hip()
    rng = np.random.default_rng(8)
    pool = Pool(dev, rng, [60, 40], 2, 64, 16)
    arr = C.c_int * 1
    i32 = _I32(dev, [0, 4, 7], [50, 30], [0, 1, 2], [0, 0], [0, 0])
    new = rng.standard_normal((2, 7, 2, 64), dtype=np.float32)
    tk, tv = _t(new[0], dev), _t(new[1], dev)
    row = N.AttnLayout(0, 64, 128)
    batch = N.KvBatch(2, 7, 4, 60, i32.ptrs[0], i32.ptrs[1])
    spare = [p for p in range(pool.num) if p not in pool.table]
    src = int(pool.table[1, 0])
    with _FreshCtx(dev) as f:
        graph, exe = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(f.stream, CAPTURE_RELAXED) == 0
        st = [f.lib.bch_kv_append(f.ctx, pool.kv, batch, _p(tk), row, _p(tv), row),
              f.lib.bch_kv_keep(f.ctx, pool.kv, 1, 0, 0, 2, 2, C.c_void_p(i32.ptrs[2]), C.c_void_p(i32.ptrs[3]),
                                C.c_void_p(i32.ptrs[4])),
              f.lib.bch_kv_copy_pages(f.ctx, pool.kv, 1, 0, 0, 1, arr(src), arr(spare[0]))]
        assert hip.hipStreamEndCapture(f.stream, C.byref(graph)) == 0 and st == [N.BCH_OK] * 3
        try:
            assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
            img = pool.pages[0]
            for lens in ([50, 30], [53, 29], [60, 40]):
                keep, to = [lens[0] - 1, lens[1] - 2], [lens[0] - 4, lens[1] - 3]
                dev.upload(i32.ptrs[1], np.array(lens, np.int32))
                dev.upload(i32.ptrs[3], np.array(keep, np.int32))
                dev.upload(i32.ptrs[4], np.array(to, np.int32))
                assert hip.hipGraphLaunch(exe, f.stream) == 0 and f.lib.bch_sync(f.ctx) == N.BCH_OK
                for b, (n, s0) in enumerate(((4, 0), (3, 4))):
                    for i in range(n):
                        j = lens[b] - n + i
                        p = img.table[b, j // 16]
                        img.k[p, :, j % 16], img.v[p, :, j % 16] = new[0, s0 + i], new[1, s0 + i]
                    a, t = keep[b], to[b]
                    for x in (img.k, img.v):
                        x[img.table[b, t // 16], :, t % 16] = x[img.table[b, a // 16], :, a % 16]
                img.k[spare[0]], img.v[spare[0]] = img.k[src], img.v[src]
                pool.check()
        finally:
            hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)


def test_keep_offsets_beyond_32_bits(dev):
    """Append, copy and keep on pages that lie beyond 2^31 floats."""
    rng = np.random.default_rng(9)
    apart, num, row = 1 << 29, 6, N.AttnLayout(0, 64, 128)
    big = [Tensor.empty([(num - 1) * apart + 2 * 16 * 64], dev) for _ in range(2)]
    i32 = _I32(dev, [[5, 4]], [0, 32], [32], [0, 3], [20, 22, 31], [17])
    table, start, length, kstart, keep, to = i32.ptrs
    lay = N.AttnLayout(apart, 16 * 64, 64)
    kv = N.KvPages(big[0].ptr, big[1].ptr, lay, lay, num, 16, 2, 64, table, 2)
    new = rng.standard_normal((2, 32, 2, 64), dtype=np.float32)
    t = [_t(x, dev) for x in new]
    dev.check(dev._lib.bch_kv_append(dev.ctx, kv, N.KvBatch(1, 32, 32, 32, start, length), _p(t[0]), row, _p(t[1]), row),
              "append")
    dev.check(dev._lib.bch_kv_keep(dev.ctx, kv, 1, 0, 0, 1, 3, *[C.c_void_p(x) for x in (kstart, keep, to)]), "keep")
    one = C.c_int * 1
    dev.check(dev._lib.bch_kv_copy_pages(dev.ctx, kv, 1, 0, 0, 1, one(4), one(0)), "copy")
    for pool, x in zip(big, new):
        x[17:20] = x[[20, 22, 31]]
        for page, rows in ((5, x[:16]), (4, x[16:]), (0, x[16:])):
            got = dev.download(pool.ptr + 4 * page * apart, 4 * 2 * 16 * 64).reshape(2, 16, 64)
            assert np.array_equal(got, rows.transpose(1, 0, 2)), page


class _Model:
    """The keys and values of every sequence and layer as lists."""

    def __init__(self, layers):
        self.keys = {}
        self.layers = layers

    def rows(self, seq, layer):
        k = [x[layer][0] if x is not None else np.full_like(self.shape, np.nan) for x in self.keys[seq]]
        v = [x[layer][1] if x is not None else np.full_like(self.shape, np.nan) for x in self.keys[seq]]
        return np.stack(k), np.stack(v), np.array([x is not None for x in self.keys[seq]])


@pytest.mark.parametrize("h,hkv,d,page", [(4, 2, 64, 16), (8, 2, 128, 8), (3, 3, 80, 5)])
def test_serving_run(dev, h, hkv, d, page):
    """Prompts, a fork, decode steps through a window, a tree of drafts verified and partly kept, eviction,
    compaction: attention is right after each."""
    rng = np.random.default_rng(d)
    layers, window, sinks = 2, 48, 3
    cache = KvCache(layers, 80, page, hkv, d, dev)
    model = _Model(layers)
    model.shape = np.zeros((hkv, d), np.float32)
    a, b = cache.new_sequence(), cache.new_sequence()
    model.keys = {a: [], b: []}

    def step(items, parents=None, w=window):
        s = cache.batch(items, parents)
        new = rng.standard_normal((layers, 2, s.total, hkv, d), dtype=np.float32)
        q = rng.standard_normal((s.total, h, d), dtype=np.float32)
        for i, (seq, n) in enumerate(items):
            at = s.start[i]
            model.keys[seq] = model.keys[seq] + [[(new[l, 0, at + x], new[l, 1, at + x]) for l in range(layers)]
                                                 for x in range(n)]
        for layer in range(layers):
            cache.append(s, layer, _t(new[layer, 0], dev), _t(new[layer, 1], dev))
            got = cache.attention(s, layer, _t(q, dev), w, sinks if w else 0).to_numpy().reshape(q.shape)
            for i, (seq, n) in enumerate(items):
                if n == 0:
                    continue
                k, v, on = model.rows(seq, layer)
                see = visible(len(on) - n, n, w, sinks if w else 0, parents[i] if parents else None)
                rows = slice(int(s.start[i]), int(s.start[i + 1]))
                scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
                want = attend(q[rows], k, v, see & on[None, :], scale)
                compare(got[rows], want, tolerance(q, k, v, scale, len(on)))
        return s

    step([(a, 100), (b, 37)])
    step([(a, 0), (b, 1)])
    c = cache.fork(a)
    model.keys[c] = list(model.keys[a])
    for _ in range(3):
        step([(c, 1), (a, 1), (b, 1)])
    step([(a, 1), (c, 2)], w=0)
    parents = [[-1, 0, 0, 1, 3, 2], [-1, -1, 1, 2]]
    s = step([(a, 6), (b, 4)], parents)
    cache.keep(s, [[0, 1, 3, 4], [1, 2]])
    for seq, n, ids in ((a, 6, [0, 1, 3, 4]), (b, 4, [1, 2])):
        old = len(model.keys[seq]) - n
        model.keys[seq] = model.keys[seq][:old] + [model.keys[seq][old + x] for x in ids]
    with pytest.raises(Exception):
        cache.keep(s, [[0], [1]])
    step([(b, 1), (c, 1), (a, 1)])
    freed = cache.evict(a, window, sinks)
    assert freed > 0
    for i, p in enumerate(cache.pages(a)):
        if p < 0:
            for j in range(i * page, (i + 1) * page):
                model.keys[a][j] = None
    step([(a, 1), (c, 1)])
    cache.free(b)
    del model.keys[b]
    assert cache.compact() > 0
    step([(a, 2), (c, 1)])
    cache.retain(c, [0, 1, 2] + list(range(60, cache.length(c))))
    model.keys[c] = model.keys[c][:3] + model.keys[c][60:]
    step([(c, 5), (a, 1)])
    cache.truncate(c, 20)
    model.keys[c] = model.keys[c][:20]
    step([(c, 1)], w=0)


def test_kv_cache_refusals_on_the_device(dev):
    cache = KvCache(1, 4, 4, 2, 64, dev)
    a = cache.new_sequence()
    s = cache.batch([(a, 2)])
    with pytest.raises(InvalidInput):
        cache.attention(s, 0, _t(np.zeros((2, 3, 64), np.float32), dev))
    empty = cache.batch([(a, 0)])
    assert cache.attention(empty, 0, Tensor.empty([0, 2, 64], dev)).shape() == [0, 2, 64]
    cache.append(empty, 0, Tensor.empty([0, 2, 64], dev), Tensor.empty([0, 2, 64], dev))
    cache.keep(empty, [[]])
