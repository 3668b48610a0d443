"""Rotary positions on the GPU against the formula in 64 bits: dense operands in both layouts, and the new tokens of a
paged cache, turned on their way into the pages."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import KvCache, Rotary, Tensor, rotary_freqs
from barracuda_amd import _native as N
from barracuda_amd.kv_cache import _I32
from tests.rotary_model import depths, turned
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip
from tests.test_gpu_kv_cache import Pool, _p, _t

pytestmark = pytest.mark.gpu


def close(got, want):
    y, bound = want
    assert got.shape == y.shape
    worst = np.max(np.abs(got - y) - bound)
    assert worst <= 0, worst


# b, h, s, d, dim, interleaved
SHAPES = [(1, 1, 1, 2, 2, False), (1, 1, 1, 2, 2, True), (2, 3, 5, 8, 8, False), (2, 3, 5, 8, 8, True), (1, 40, 1, 128, 128, False),
          (3, 4, 17, 64, 64, True), (2, 5, 33, 80, 40, False), (2, 5, 33, 80, 40, True), (1, 2, 70, 96, 42, False),
          (2, 2, 9, 33, 20, True), (1, 3, 6, 257, 256, False), (1, 2, 3, 1030, 1028, True), (1, 1, 4, 4096, 2048, False),
          (1, 70, 2, 64, 16, False), (4, 1, 700, 32, 32, False), (1, 2, 2, 12, 4, False)]


@pytest.mark.parametrize("heads_last", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("b,h,s,d,dim,interleaved", SHAPES)
def test_dense(dev, b, h, s, d, dim, interleaved, inverse, heads_last):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((b, s, h, d) if heads_last else (b, h, s, d), dtype=np.float32)
    r = Rotary(d, dim=dim, interleaved=interleaved, scale=1.25)
    first = 1000
    got = _t(x, dev).rotary(r, first=first, inverse=inverse, heads_last=heads_last).to_numpy()
    pos = first + np.arange(s)
    close(got, turned(x, pos[None, :, None] if heads_last else pos[None, None], r.freqs, dim, interleaved, 1.25, inverse))


@pytest.mark.parametrize("top", [1, 4096, 2**20, 2**31 - 1])
def test_far_and_negative_positions(dev, top):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 50, 2, 64), dtype=np.float32)
    pos = rng.integers(-top - 1, top, (3, 50), endpoint=True)
    pos[0, :2] = -top - 1, top
    r = Rotary(64, interleaved=True)
    got = _t(x, dev).rotary(r, positions=pos, heads_last=True).to_numpy()
    # an angle of 2^31 in 64 bits is off by 2^-22: its product is rounded here and there alike
    close(got, turned(x, pos[:, :, None], r.freqs, 64, True, 1.0))


def test_fast_frequencies_and_zero(dev):
    """Angles far beyond 2^31 quarter turns stay what they are in 64 bits; frequency 0 leaves the pair, scale 0 nothing."""
    x = np.random.default_rng(3).standard_normal((1, 2, 40, 8), dtype=np.float32)
    f = [0.0, 3.0, 40.0, 1e-9]
    for scale in (1.0, 0.0, -2.0):
        r = Rotary(8, freqs=f, scale=scale)
        close(_t(x, dev).rotary(r, first=10**6).to_numpy(), turned(x, 10**6 + np.arange(40), np.array(f), 8, False, scale))


def test_special_values_stay_in_their_pairs(dev):
    x = np.ones((1, 1, 3, 16), np.float32)
    x[0, 0, 0, 1], x[0, 0, 1, 9], x[0, 0, 2, 15] = np.nan, np.inf, -np.inf
    got = _t(x, dev).rotary(Rotary(16), first=5).to_numpy()
    bad = ~np.isfinite(got)
    want = np.zeros_like(bad)
    want[0, 0, 0, [1, 9]] = want[0, 0, 1, [1, 9]] = want[0, 0, 2, [7, 15]] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_transpose(dev, interleaved):
    """<turn(x), y> = <x, inverse(y)>, the gradient's definition; and a difference of two turns is the turn of the difference."""
    rng = np.random.default_rng(4)
    x, y, dx = (rng.standard_normal((2, 3, 21, 24), dtype=np.float32) for _ in range(3))
    r = Rotary(24, dim=16, interleaved=interleaved, scale=1.5)
    t = lambda a, inv=False: _t(a, dev).rotary(r, first=77, inverse=inv).to_numpy().astype(np.float64)
    left, right = (t(x) * y).sum(), (x * t(y, True)).sum()
    # sums of n products whose factors are off by BOUND * 1.5 * (|a| + |b|)
    slack = 2 * 5 * 2.0**-24 * 1.5 * 2 * (np.abs(x).max() * np.abs(y).sum() + np.abs(y).max() * np.abs(x).sum())
    assert abs(left - right) <= slack
    h = np.float32(2.0**-3)
    diff = (t(x + h * dx) - t(x - h * dx)) / (2 * float(h))
    want, _ = turned(dx, 77 + np.arange(21), r.freqs, 16, interleaved, 1.5)
    assert np.max(np.abs(diff - want)) <= 2.0**-24 * 100 * 2 / (2 * float(h)) * (np.abs(x).max() + np.abs(dx).max())


@pytest.mark.parametrize("misalign", [0, 1])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_strides_and_in_place(dev, pad, misalign):
    b, h, s, d = 2, 3, 19, 32
    rng = np.random.default_rng(5)
    w = d + pad
    whole = rng.standard_normal((misalign + b * h * s * w,), dtype=np.float32)
    t = _t(whole, dev)
    lay = N.AttnLayout(h * s * w, s * w, w)
    r = Rotary(d, dim=24)
    ptr = C.c_void_p(t.ptr + 4 * misalign)
    dev.check(dev._lib.bch_rotary(dev.ctx, b, h, s, d, r._plan, 0, 3, None, ptr, lay, ptr, lay), "rotary")
    got = t.to_numpy()
    x, y = (a[misalign:].reshape(b, h, s, w) for a in (whole, got))
    close(y[..., :d], turned(x[..., :d], 3 + np.arange(s), r.freqs, 24, False, 1.0))
    assert np.array_equal(y[..., d:], x[..., d:]) and np.array_equal(got[:misalign], whole[:misalign])
    other = N.AttnLayout(h * s * w, w, h * w)
    st = dev._lib.bch_rotary(dev.ctx, b, h, s, d, r._plan, 0, 3, None, ptr, lay, ptr, other)
    assert st == N.BCH_E_INVALID


def test_one_head_read_by_all(dev):
    """A head stride of 0: every head of o gets the same turned row."""
    x = np.random.default_rng(6).standard_normal((2, 1, 11, 16), dtype=np.float32)
    t, o = _t(x, dev), Tensor.empty([2, 5, 11, 16], dev)
    r = Rotary(16)
    dev.check(dev._lib.bch_rotary(dev.ctx, 2, 5, 11, 16, r._plan, 0, 0, None, _p(t), N.AttnLayout(176, 0, 16), _p(o),
                                  N.AttnLayout(880, 176, 16)), "rotary")
    close(o.to_numpy(), turned(np.repeat(x, 5, 1), np.arange(11), r.freqs, 16, False, 1.0))


def test_empty(dev):
    r = Rotary(8)
    for shape in ([0, 2, 3, 8], [2, 0, 3, 8], [2, 2, 0, 8]):
        assert Tensor.empty(shape, dev).rotary(r).shape() == shape


# ---- the new tokens of a paged cache ----

# heads, kv heads, d, dim, interleaved, page, pad, misalign, slots
APPEND = [(4, 2, 64, 64, False, 16, 0, 0, False), (1, 1, 4, 2, True, 3, 0, 0, False), (8, 8, 128, 128, True, 16, 0, 0, False),
          (6, 3, 80, 40, False, 24, 4, 0, True), (5, 5, 33, 20, True, 5, 0, 0, False), (2, 1, 64, 32, False, 8, 0, 1, False),
          (32, 2, 48, 48, True, 1, 3, 0, True), (0, 2, 64, 64, False, 16, 0, 0, False), (2, 2, 300, 300, False, 7, 0, 0, True)]


def _append(dev, pool, lens, news, h, r, rng, parents=None, total=None, max_new=None, extra=0):
    start = np.concatenate([[0], np.cumsum(news)])
    rows = int(start[-1]) + extra
    total = rows if total is None else total
    w = pool.d + pool.pad
    i32 = _I32(dev, start, lens, [p for t in parents for p in t] if parents is not None else [])
    batch = N.KvBatch(len(lens), total, max(news) if max_new is None else max_new, max(lens), i32.ptrs[0], i32.ptrs[1])
    shift = np.zeros(pool.misalign, np.float32)
    new = rng.standard_normal((2, rows, pool.hkv, w), dtype=np.float32)
    q = rng.standard_normal((rows, max(h, 1), w), dtype=np.float32)
    tk, tv, tq = (_t(np.concatenate([shift, x.reshape(-1)]), dev) for x in (*new, q))
    to = _t(np.full(pool.misalign + q.size, 7.0, np.float32), dev)
    row, q_row = N.AttnLayout(0, w, pool.hkv * w), N.AttnLayout(0, w, max(h, 1) * w)
    p = [C.c_void_p(t.ptr + 4 * pool.misalign) for t in (tq, to, tk, tv)]
    dev.check(dev._lib.bch_kv_append_rotary(dev.ctx, pool.kv, batch, C.c_void_p(i32.ptrs[2]) if parents is not None else None,
                                            r._plan, h, p[0], q_row, p[1], q_row, p[2], row, p[3], row), "append")
    out = to.to_numpy()[pool.misalign:].reshape(q.shape)
    seen = np.zeros(rows, bool)
    img = pool.pages[0]
    got = {x: t.to_numpy() for x, t in (("k", pool.tk), ("v", pool.tv))}
    bounds = np.zeros_like(img.k, dtype=np.float64)
    wide = img.k.astype(np.float64)
    for b, (length, n) in enumerate(zip(lens, news)):
        depth = depths(parents[b]) if parents is not None else list(range(n))
        for i in range(min(n, batch.max_new)):
            x = start[b] + i
            if x >= total:
                continue
            seen[x] = True
            pos = length - n + depth[i]
            if h:
                close(out[x, :, :pool.d], turned(q[x, :, :pool.d], pos, r.freqs, r.dim, r.interleaved, r.scale))
            j = length - n + i
            page = pool.table[b, j // pool.page] if j >= 0 else -1
            if 0 <= page < pool.num:
                at = (page, slice(None), j % pool.page)
                wide[at], bounds[at] = turned(new[0, x, :, :pool.d], pos, r.freqs, r.dim, r.interleaved, r.scale)
                img.v[at] = new[1, x, :, :pool.d]
    # rows that are no new token's, and padding between rows, are as before
    assert h == 0 or np.all(out[~seen] == 7.0)
    assert np.all(out[..., pool.d:] == 7.0)
    keep = img.k
    img.k = wide.astype(np.float32)
    want = pool._put([img.k]).to_numpy()
    img.k = bounds.astype(np.float32)
    slack = pool._put([img.k]).to_numpy()
    slack[want == 5.0] = 0.0
    # the image itself is rounded once, its bound once
    assert np.all(np.abs(got["k"] - want) <= slack * (1 + 2.0**-20) + 2.0**-24 * np.abs(want) * (slack > 0))
    img.k = keep
    assert np.array_equal(got["v"], pool._put([img.v]).to_numpy())


@pytest.mark.parametrize("h,hkv,d,dim,interleaved,page,pad,misalign,slots", APPEND)
@pytest.mark.parametrize("lens,news", [([1], [1]), ([40, 7, 33, 0, 9], [1, 0, 33, 0, 1]), ([100, 61], [59, 61]), ([3, 20], [5, 4])])
def test_append(dev, lens, news, h, hkv, d, dim, interleaved, page, pad, misalign, slots):
    rng = np.random.default_rng(7)
    pool = Pool(dev, rng, lens, hkv, d, page, 1, slots, pad, misalign)
    _append(dev, pool, lens, news, h, Rotary(d, dim=dim, interleaved=interleaved, scale=1.1), rng)


@pytest.mark.parametrize("h,hkv,d,dim,interleaved,page,pad,misalign,slots", APPEND[:5])
@pytest.mark.parametrize("news", [[1], [7, 0, 128], [2, 64, 33]])
def test_append_trees(dev, news, h, hkv, d, dim, interleaved, page, pad, misalign, slots):
    rng = np.random.default_rng(8)
    lens = [n + int(rng.integers(0, 50)) for n in news]
    trees = [[-1 if i == 0 else int(rng.integers(-1, i)) for i in range(n)] for n in news]
    if len(news) > 2:
        trees[2] = list(range(-1, news[2] - 1))  # a chain
        trees[0][1] = 5  # not below its draft: a child of the last committed token
    pool = Pool(dev, rng, lens, hkv, d, page, 1, slots, pad, misalign)
    _append(dev, pool, lens, news, h, Rotary(d, dim=dim, interleaved=interleaved), rng, trees)


# room for more rows; rows beyond max_new stay; a longest length that none has
@pytest.mark.parametrize("kwargs", [{}, {"extra": 5}, {"max_new": 7}, {"max_new": 2**31 - 1}])
def test_append_pages_not_held_and_rows_behind(dev, kwargs):
    rng = np.random.default_rng(9)
    lens, news = [20, 40, 6], [20, 9, 6]
    pool = Pool(dev, rng, lens, 2, 64, 8)
    pool.table[0, 2], pool.table[1, [1, 4]] = -1, [pool.num, 2**30]
    pool.i32 = _I32(dev, pool.table)
    pool.kv.table = pool.i32.ptrs[0]
    _append(dev, pool, lens, news, 4, Rotary(64), rng, **kwargs)


def test_append_beyond_a_grid(dev):
    """Batch times the longest chunk's tiles is beyond a grid: the rows that there are look for their sequences."""
    rng = np.random.default_rng(10)
    nb = 1 << 18
    lens, news = np.zeros(nb, np.int64), np.zeros(nb, np.int64)
    some = [0, 5, 6, 70000, nb - 2, nb - 1]
    for b, (length, n) in zip(some, [(900, 900), (30, 1), (1, 1), (3, 5), (70, 64), (4, 2)]):
        lens[b], news[b] = length, n
    small = Pool(dev, rng, [int(lens[b]) for b in some], 2, 32, 16)
    table = np.full((nb, small.table.shape[1]), -1, np.int32)
    table[some] = small.table
    whole = _I32(dev, table)
    start = np.concatenate([[0], np.cumsum(news)])
    total, h = int(start[-1]), 3
    for trees in (False, True):
        cut = min(128, total) if trees else total
        i32 = _I32(dev, start, lens, np.repeat(-1, total))
        kv = N.KvPages(small.tk.ptr, small.tv.ptr, small.kv.k_layout, small.kv.v_layout, small.num, 16, 2, 32, whole.ptrs[0],
                       table.shape[1])
        batch = N.KvBatch(nb, total, cut, 900, i32.ptrs[0], i32.ptrs[1])
        q = rng.standard_normal((total, h, 32), dtype=np.float32)
        k, v = rng.standard_normal((2, total, 2, 32), dtype=np.float32)
        tq, tk, tv, to = _t(q, dev), _t(k, dev), _t(v, dev), _t(np.full_like(q, 7.0), dev)
        row, q_row = N.AttnLayout(0, 32, 64), N.AttnLayout(0, 32, 96)
        r = Rotary(32)
        dev.check(dev._lib.bch_kv_append_rotary(dev.ctx, kv, batch, C.c_void_p(i32.ptrs[2]) if trees else None, r._plan, h,
                                                _p(tq), q_row, _p(to), q_row, _p(tk), row, _p(tv), row), "append")
        out, pk, pv = to.to_numpy(), small.tk.to_numpy().reshape(small.num, 2, 16, 32), small.tv.to_numpy().reshape(small.num, 2, 16, 32)
        for x, b in enumerate(some):
            for i in range(news[b]):
                row_i = start[b] + i
                if i >= cut:
                    assert np.all(out[row_i] == 7.0)
                    continue
                j = int(lens[b] - news[b] + i)
                pos = int(lens[b] - news[b]) if trees else j
                close(out[row_i], turned(q[row_i], pos, r.freqs, 32, False, 1.0))
                if j >= 0:
                    p = small.table[x, j // 16]
                    close(pk[p, :, j % 16], turned(k[row_i], pos, r.freqs, 32, False, 1.0))
                    assert np.array_equal(pv[p, :, j % 16], v[row_i])


def test_append_in_place_equals_apart(dev):
    rng = np.random.default_rng(11)
    lens, news = [50, 9], [50, 1]
    q = rng.standard_normal((51, 4, 64), dtype=np.float32)
    k = rng.standard_normal((51, 2, 64), dtype=np.float32)
    r, outs = Rotary(64), []
    for same in (False, True):
        pool = Pool(dev, np.random.default_rng(1), lens, 2, 64, 16)
        i32 = _I32(dev, [0, 50, 51], lens)
        tq, tk = _t(q, dev), _t(k, dev)
        to = tq if same else Tensor.empty([51, 4, 64], dev)
        q_row, row = N.AttnLayout(0, 64, 256), N.AttnLayout(0, 64, 128)
        dev.check(dev._lib.bch_kv_append_rotary(dev.ctx, pool.kv, N.KvBatch(2, 51, 50, 50, *i32.ptrs), None, r._plan, 4, _p(tq),
                                                q_row, _p(to), q_row, _p(tk), row, _p(tk), row), "append")
        outs.append((to.to_numpy(), pool.tk.to_numpy()))
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[1][1])


def test_cache_with_turned_keys_attends_to_distances(dev):
    """KvCache.append_rotary then attention, token by token and with drafts: the same as one call over the whole sequence
    with positions shifted, for only distances count."""
    rng = np.random.default_rng(12)
    h, hkv, d, n = 4, 2, 32, 23
    q, k, v = (rng.standard_normal((n, x, d), dtype=np.float32) for x in (h, hkv, hkv))
    r = Rotary(d)
    c = KvCache(1, 16, 4, hkv, d, dev)
    a, rows = c.new_sequence(), []
    for lo, hi in ((0, 9), (9, 10), (10, 11), (11, 17)):
        step = c.batch([(a, hi - lo)])
        turned_q = c.append_rotary(step, 0, r, *(_t(x[lo:hi], dev) for x in (q, k, v)))
        rows.append(c.attention(step, 0, turned_q).to_numpy())
    # two branches of drafts, the first of them the sequence's own tokens
    step = c.batch([(a, 7)], parents=[[-1, 0, -1, 1, 3, 4, 5]])
    order = [17, 18, 3, 19, 20, 21, 22]
    turned_q = c.append_rotary(step, 0, r, *(_t(x[order], dev) for x in (q, k, v)))
    rows.append(c.attention(step, 0, turned_q).to_numpy()[[0, 1, 3, 4, 5, 6]])
    got = np.concatenate(rows)
    # whole: [1, H, S, D] operands, from position 5000 on
    tq, tk = (_t(x.transpose(1, 0, 2)[None].copy(), dev).rotary(r, first=5000) for x in (q, k))
    want = tq.sliding_window_attention(tk, _t(v.transpose(1, 0, 2)[None].copy(), dev), 0).to_numpy()[0].transpose(1, 0, 2)
    # scores of up to 40 whose operands are off by BOUND (|a| + |b|) twice: relative weights off by 40 * 4 * 5 * 2^-24
    scores = np.abs(np.einsum("ihd,jhd->hij", np.abs(q), np.repeat(np.abs(k), h // hkv, 1))).max() / np.sqrt(d)
    assert np.max(np.abs(got - want)) <= 2 * scores * 4 * 5 * 2.0**-24 * np.abs(v).max() * 2


def test_captured_append_reads_lengths_at_replay(dev):
    with _FreshCtx(dev) as f:
        _captured(_hip(), f)


def _captured(hip, f):
    lens, h, hkv, d, page = [5, 9], 4, 2, 32, 8
    rng = np.random.default_rng(13)
    k = np.zeros((8, hkv, page, d), np.float32)

    def up(x):
        p = C.c_void_p()
        assert f.lib.bch_alloc(f.ctx, x.nbytes, C.byref(p)) == 0
        assert f.lib.bch_upload(f.ctx, p, x.ctypes.data_as(C.c_void_p), x.nbytes) == 0
        return p
    q, nk, nv = (rng.standard_normal((2, x, d), dtype=np.float32) for x in (h, hkv, hkv))
    freqs = rotary_freqs(d)
    pq, pk, pv, po, kk, kv = up(q), up(nk), up(nv), up(q), up(k), up(k)
    pf, pt = up(freqs), up(np.array([[0, 1, 2, 3], [4, 5, 6, 7]], np.int32))
    ps, pl = up(np.array([0, 1, 2], np.int32)), up(np.array(lens, np.int32))
    lay = N.AttnLayout(hkv * page * d, page * d, d)
    pages = N.KvPages(kk.value, kv.value, lay, lay, 8, page, hkv, d, pt.value, 4)
    batch = N.KvBatch(2, 2, 1, 9, ps.value, pl.value)
    plan = N.Rotary(d, 0, 1.0, pf.value)
    row, q_row = N.AttnLayout(0, d, hkv * d), N.AttnLayout(0, d, h * d)
    call = lambda: f.lib.bch_kv_append_rotary(f.ctx, pages, batch, None, plan, h, pq, q_row, po, q_row, pk, row, pv, row)
    stream = f.stream
    assert hip.hipStreamBeginCapture(stream, CAPTURE_RELAXED) == 0
    st = call()
    graph, ex = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0 and st == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for now in ([5, 9], [6, 10], [1, 32], [17, 2]):
        a = np.array(now, np.int32)
        assert f.lib.bch_upload(f.ctx, pl, a.ctypes.data_as(C.c_void_p), a.nbytes) == 0
        assert hip.hipGraphLaunch(ex, stream) == 0 and f.lib.bch_sync(f.ctx) == 0
        out, got = np.empty_like(q), np.empty_like(k)
        assert f.lib.bch_download(f.ctx, out.ctypes.data_as(C.c_void_p), po, out.nbytes) == 0
        assert f.lib.bch_download(f.ctx, got.ctypes.data_as(C.c_void_p), kk, got.nbytes) == 0
        for b, length in enumerate(now):
            close(out[b], turned(q[b], length - 1, freqs, d, False, 1.0))
            close(got[4 * b + (length - 1) // page, :, (length - 1) % page], turned(nk[b], length - 1, freqs, d, False, 1.0))
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
