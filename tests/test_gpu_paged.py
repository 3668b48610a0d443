"""Attention with a window and sinks, over dense operands and over a paged cache, and trees of drafts, against
the plain form in 64 bits: edges of key blocks, pages and windows, ragged batches, strides, masks that leave a
row empty, values that no row may see, captured calls."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Tensor
from barracuda_amd import _native as N
from barracuda_amd.error import UnsupportedOperation
from barracuda_amd.kv_cache import _I32
from tests.kv_model import Pages, attend, visible
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip

pytestmark = pytest.mark.gpu


def tolerance(q, k, v, scale, keys):
    """Four standard deviations of a random walk of roundings of 2^-24 each: a score's D + 2 additions of terms
    that sum to S in magnitude, which enter the weights of numerator and denominator, and the `keys` additions
    of a weighted mean; times the largest value."""
    # the planted values apart, which no compared row sees
    fin = lambda x: np.abs(np.where(np.isfinite(x) & (np.abs(x) < 1e30), x, 0.0)).astype(np.float64)
    d = q.shape[-1]
    s = abs(scale) * np.sqrt((fin(q) ** 2).sum(-1).max()) * np.sqrt((fin(k) ** 2).sum(-1).max())
    return 4 * 2.0**-24 * fin(v).max() * (2 * np.sqrt(d + 2) * s + np.sqrt(max(keys, 1)) + 8)


class Case:
    """A call over scattered pages with everything it needs in HBM."""

    def __init__(self, dev, lens, news, h, hkv, d, page, window=0, sinks=0, parents=None, seed=0, row_pad=0, slots=False,
                 fill=None, misalign=0, scale=None, max_new=None, tail_rows=2):
        rng = np.random.default_rng(seed + 1000 * d + 10 * page + sum(lens))
        self.dev, self.lens, self.news, self.h, self.hkv, self.d = dev, lens, news, h, hkv, d
        self.window, self.sinks, self.parents = window, sinks, parents
        self.scale = scale if scale is not None else float(1.0 / np.sqrt(d))
        self.pool = Pages(rng, lens, hkv, d, page, fill=fill)
        self.start = np.concatenate([[0], np.cumsum(news)])
        self.total = int(self.start[-1])
        self.rows = self.total + tail_rows  # rows behind the last sequence
        self.q = rng.standard_normal((self.rows, h, d), dtype=np.float32)
        self.page, self.slots, self.row_pad, self.misalign = page, slots, row_pad, misalign
        self.max_new = max(news) if max_new is None else max_new
        self.upload()

    def _put(self, x):
        """x's floats, misalign floats behind a 16-byte boundary."""
        t = Tensor.from_data(np.concatenate([np.zeros(self.misalign, np.float32), x.reshape(-1)]),
                             [x.size + self.misalign], self.dev)
        return t, t.ptr + 4 * self.misalign

    def upload(self):
        p, d, pad = self.pool, self.d, self.row_pad
        def store(x):  # [pages, Hkv, page, D], or with heads inside slots; rows pad floats apart
            y = np.full(x.shape[:3] + (d + pad,), np.nan, np.float32)
            y[..., :d] = x
            return np.ascontiguousarray(y.transpose(0, 2, 1, 3)) if self.slots else y
        self.tk, pk = self._put(store(p.k))
        self.tv, pv = self._put(store(p.v))
        w = d + pad
        lay = (N.AttnLayout(self.hkv * self.page * w, w, self.hkv * w) if self.slots
               else N.AttnLayout(self.hkv * self.page * w, self.page * w, w))
        flat = [] if self.parents is None else [x for t in self.parents for x in t]
        self.i32 = _I32(self.dev, self.start, self.lens, p.table, flat)
        self.kv = N.KvPages(pk, pv, lay, lay, p.num, self.page, self.hkv, d, self.i32.ptrs[2], p.table.shape[1])
        self.batch = N.KvBatch(len(self.lens), self.total, self.max_new, max(self.lens + [0]), self.i32.ptrs[0],
                               self.i32.ptrs[1])
        y = np.full((self.rows, self.h, w), np.nan, np.float32)
        y[..., :d] = self.q
        self.tq, self.pq = self._put(y)
        self.to, self.po = self._put(np.full((self.rows, self.h, w), 7.0, np.float32))
        self.row = N.AttnLayout(0, w, self.h * w)

    def call(self, lib, ctx):
        parent = C.c_void_p(self.i32.ptrs[3]) if self.parents is not None else None
        return lib.bch_sdpa_paged(ctx, self.kv, self.batch, self.h, self.scale, self.window, self.sinks, parent,
                                  C.c_void_p(self.pq), self.row, C.c_void_p(self.po), self.row)

    def output(self):
        out = self.to.to_numpy()[self.misalign:].reshape(self.rows, self.h, self.d + self.row_pad)
        assert np.all(out[..., self.d:] == 7.0), "padding written"
        assert np.all(out[self.total:] == 7.0), "rows behind the last sequence written"
        return out[:self.total, :, :self.d]

    def want(self):
        out = np.zeros((self.total, self.h, self.d))
        for b, (length, n) in enumerate(zip(self.lens, self.news)):
            if n == 0:
                continue
            first = length - n
            see = visible(first, n, self.window, self.sinks, self.parents[b] if self.parents is not None else None)
            (k, on), (v, _) = self.pool.keys(b, length, self.pool.k), self.pool.keys(b, length, self.pool.v)
            rows = slice(int(self.start[b]), int(self.start[b + 1]))
            out[rows] = attend(self.q[rows], k, v, see & on[None, :], self.scale)
        return out

    def check(self):
        self.dev.check(self.call(self.dev._lib, self.dev.ctx), "attention")
        got, want = self.output(), self.want()
        compare(got, want, tolerance(self.q, self.pool.k, self.pool.v, self.scale, max(self.lens)))
        self.dev.check(self.call(self.dev._lib, self.dev.ctx), "attention")
        assert np.array_equal(got, self.output(), equal_nan=True), "not deterministic"
        return got


def compare(got, want, tol):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fin = np.isfinite(want)
    err = np.abs(got[fin] - want[fin]).max() if fin.any() else 0.0
    assert err <= tol, f"error {err:.3g} above {tol:.3g}"


# ---- one new token a sequence, chunks, whole prompts ------------------------------------------


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 0), (33, 4), (100, 40), (5000, 3)])
@pytest.mark.parametrize("lens,h,hkv,d,page", [
    ([1], 1, 1, 64, 16), ([300, 1, 17, 64], 8, 8, 64, 16), ([1000, 1023, 1024, 1025, 31], 8, 2, 128, 32),
    ([130, 257], 15, 3, 80, 24), ([97, 401], 16, 1, 96, 7), ([512, 333], 6, 2, 36, 1), ([200, 129], 40, 1, 128, 256)])
def test_one_token(dev, lens, h, hkv, d, page, window, sinks):
    print(f"one lens={lens} h={h} hkv={hkv} d={d} page={page} window={window} sinks={sinks}", flush=True)
    Case(dev, lens, [1] * len(lens), h, hkv, d, page, window, sinks).check()


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 0), (64, 5), (200, 33), (70, 4000)])
@pytest.mark.parametrize("lens,news,h,hkv,d,page", [
    ([5], [5], 1, 1, 32, 4), ([70, 33, 400], [70, 1, 31], 4, 2, 64, 16), ([300, 290, 8, 0], [129, 290, 0, 0], 8, 2, 128, 32),
    ([260, 513], [257, 300], 3, 3, 80, 24), ([150, 611], [65, 2], 12, 2, 96, 128), ([90, 200], [90, 200], 9, 1, 48, 5)])
def test_chunks(dev, lens, news, h, hkv, d, page, window, sinks):
    print(f"chunks lens={lens} news={news} h={h} hkv={hkv} d={d} page={page} window={window} sinks={sinks}", flush=True)
    Case(dev, lens, news, h, hkv, d, page, window, sinks).check()


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("h,hkv", [(2, 2), (4, 1)])
def test_every_block_edge(dev, n, h, hkv):
    """Rows and keys on either side of the blocks that the kernels use."""
    for more in (0, 1, 40):
        print(f"edge n={n} more={more} h={h} hkv={hkv}", flush=True)
        Case(dev, [n + more, 2 * n], [n, n], h, hkv, 128, 16, 24, 2).check()


@pytest.mark.parametrize("d", [1, 2, 3, 5, 8, 30, 33, 63, 65, 100, 127, 130, 192, 256, 257, 300, 600, 1024])
def test_every_width(dev, d):
    for lens, news in (([70, 9], [1, 1]), ([90, 41], [40, 17])):
        print(f"width d={d} lens={lens} news={news}", flush=True)
        Case(dev, lens, news, 4, 2, d, 16, 30, 3).check()


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("row_pad,misalign", [(0, 0), (4, 0), (3, 0), (0, 1), (4, 2)])
@pytest.mark.parametrize("lens,news", [([333, 40], [1, 1]), ([333, 140], [100, 140])])
def test_strides_and_alignment(dev, lens, news, row_pad, misalign, slots):
    for d in (64, 128, 50):
        print(f"strides pad={row_pad} misalign={misalign} slots={slots} news={news} d={d}", flush=True)
        Case(dev, lens, news, 6, 2, d, 16, 100, 2, row_pad=row_pad, misalign=misalign, slots=slots).check()


def test_wide_groups_and_many_sequences(dev):
    Case(dev, [300, 77], [3, 20], 128, 1, 64, 16, 50, 1).check()
    lens = [1 + 7 * (i % 50) for i in range(300)]
    Case(dev, lens, [min(n, 1 + i % 3) for i, n in enumerate(lens)], 4, 2, 32, 8, 40, 2).check()


def test_long_sequences_and_a_long_row(dev):
    """Many splits of the keys: one long sequence beside short ones, with and without a window."""
    for window, sinks in ((0, 0), (3000, 4)):
        Case(dev, [20011, 5, 777], [1, 1, 1], 8, 2, 128, 64, window, sinks).check()
        Case(dev, [9000, 200], [40, 70], 4, 1, 64, 64, window, sinks).check()


def test_more_rows_than_keys(dev):
    """Rows that stand before the first key see nothing and give zeros."""
    got = Case(dev, [3, 0, 5], [6, 4, 5], 4, 2, 64, 16, 2, 1).check()
    assert np.all(got[:3] == 0) and np.all(got[6:10] == 0)


def test_max_new_leaves_the_rows_beyond(dev):
    c = Case(dev, [50, 60], [20, 30], 4, 2, 64, 16, max_new=20)
    dev.check(c.call(dev._lib, dev.ctx), "attention")
    got, want = c.output(), c.want()
    tol = tolerance(c.q, c.pool.k, c.pool.v, c.scale, 60)
    compare(got[:40], want[:40], tol)
    assert np.all(got[40:] == 7.0)


def test_empty_calls(dev):
    c = Case(dev, [5], [2], 2, 2, 32, 4)
    for f in ("B", "total", "max_new"):
        b = N.KvBatch.from_buffer_copy(c.batch)
        setattr(b, f, 0)
        old, c.batch = c.batch, b
        dev.check(c.call(dev._lib, dev.ctx), "attention")
        assert np.all(c.to.to_numpy() == 7.0)
        c.batch = old


# ---- pages that are not held, values that no row may see ----------------------------------------


@pytest.mark.parametrize("news", [[1, 1], [30, 200]])
def test_pages_not_held(dev, news):
    """Table entries outside the pool are keys that nobody sees; a sequence without any gives zeros."""
    c = Case(dev, [400, 300], news, 4, 2, 64, 16, 0, 0)
    c.pool.table[0, [0, 3, 7, 24]] = [-1, c.pool.num, 2**31 - 1, -2**31]
    c.upload()
    c.check()
    c.pool.table[1, :] = -1
    c.upload()
    got = c.check()
    assert np.all(got[news[0]:] == 0)


def test_a_length_beyond_the_table_counts_as_the_tables(dev):
    c = Case(dev, [64, 40], [1, 1], 4, 2, 64, 16)
    c.i32 = _I32(dev, c.start, [1000, 40], c.pool.table)
    c.kv.table, c.batch.start, c.batch.len = c.i32.ptrs[2], c.i32.ptrs[0], c.i32.ptrs[1]
    dev.check(c.call(dev._lib, dev.ctx), "attention")
    compare(c.output(), c.want(), tolerance(c.q, c.pool.k, c.pool.v, c.scale, 64))


def test_starts_are_clamped_to_the_rows(dev):
    c = Case(dev, [64, 40], [3, 2], 4, 2, 64, 16)
    for start in ([-5, 3, 400], [0, 3, 2**31 - 1], [4, 2, -7]):
        c.i32 = _I32(dev, start, c.lens, c.pool.table)
        c.kv.table, c.batch.start, c.batch.len = c.i32.ptrs[2], c.i32.ptrs[0], c.i32.ptrs[1]
        dev.check(c.call(dev._lib, dev.ctx), "attention")
        c.output()  # padding and the rows behind stay


def test_starts_that_do_not_ascend_stay_in_bounds(dev):
    """Keys split over workgroups and starts that name no sequence's rows: nothing outside the rows is written."""
    for news, starts in (([3, 2, 4], ([0, 7, 3, 9], [9, 0, 0, 5], [5, 2, 2**31 - 1, 1])),
                         ([40, 100, 70], ([100, 0, 150, 30], [210, 1, 0, 90], [-8, 150, 10, 2**31 - 1]))):
        c = Case(dev, [3000, 2500, 1800], news, 8, 2, 128, 16)
        c.check()
        for start in starts:
            c.i32 = _I32(dev, start, c.lens, c.pool.table)
            c.kv.table, c.batch.start, c.batch.len = c.i32.ptrs[2], c.i32.ptrs[0], c.i32.ptrs[1]
            dev.check(c.call(dev._lib, dev.ctx), "attention")
            c.output()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max])
@pytest.mark.parametrize("lens,news,h,hkv,d,page", [
    ([170, 45], [1, 1], 4, 2, 64, 16), ([170, 45, 300], [50, 45, 130], 4, 2, 128, 16), ([200], [200], 3, 3, 80, 24)])
def test_values_behind_the_mask_do_not_reach_a_row(dev, lens, news, h, hkv, d, page, bad):
    """Everything in the pool that is not a key is `bad`, and so are keys that some rows see and others do not."""
    c = Case(dev, lens, news, h, hkv, d, page, 20, 2, fill=bad)
    compare(c.check(), c.want(), tolerance(c.q, c.pool.k, c.pool.v, c.scale, max(lens)))
    for b, (length, n) in enumerate(zip(lens, news)):
        for j in (length - 1, length - min(n, 30), max(0, length - 25), 0):
            if j > 1 or n > 60:
                c.pool.v[c.pool.table[b, j // page], 0, j % page, ::3] = bad
                c.pool.k[c.pool.table[b, j // page], hkv - 1, j % page, 1] = bad if n > 1 else 1.0
    c.upload()
    if np.isfinite(bad):  # scores of the type's largest numbers: only where they are not seen can be told
        c.dev.check(c.call(dev._lib, dev.ctx), "attention")
        got = c.output()
        seen = np.zeros(c.total, bool)
        for b, (length, n) in enumerate(zip(lens, news)):
            see = visible(length - n, n, 20, 2)
            k, _ = c.pool.keys(b, length, c.pool.k)
            v, _ = c.pool.keys(b, length, c.pool.v)
            hot = (np.abs(k).max((1, 2)) == bad) | (np.abs(v).max((1, 2)) == bad)
            seen[c.start[b]:c.start[b + 1]] = (see & hot[None, :]).any(1)
        want = c.want()
        compare(got[~seen], want[~seen], tolerance(c.q, c.pool.k, c.pool.v, c.scale, max(lens)))
    else:
        c.check()


def test_extreme_queries(dev):
    """A NaN or infinite query is NaN in its own row and nowhere else; scores far above the rest win alone."""
    for news in ([2, 3], [60, 33]):
        c = Case(dev, [200, 90], news, 4, 2, 64, 16, 40, 2)
        c.q[0, 1, 3] = np.nan
        c.q[c.total - 1, 2, 0] = np.inf
        c.q[c.total // 2, 0] = 1e18
        c.upload()
        dev.check(c.call(dev._lib, dev.ctx), "attention")
        got, want = c.output(), c.want()
        rows = np.ones(c.total, bool)
        rows[[0, c.total - 1, c.total // 2]] = False
        compare(got[rows], want[rows], tolerance(c.q[:c.total][rows], c.pool.k, c.pool.v, c.scale, 200))
        assert np.all(np.isnan(got[0, 1])) and np.all(np.isnan(got[c.total - 1, 2]))
        assert np.all(np.isfinite(got[0, [0, 2, 3]]))
        assert np.all(np.isfinite(got[c.total // 2]))


# ---- trees of drafts -------------------------------------------------------------------------------


def _tree(rng, n, deep):
    return [-1 if i == 0 or rng.random() < 0.15 else int(rng.integers(max(0, i - 2) if deep else 0, i)) for i in range(n)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 0), (2, 300), (40, 4)])
@pytest.mark.parametrize("lens,news,h,hkv,d,page", [
    ([1], [1], 2, 2, 64, 16), ([9, 8], [8, 8], 4, 4, 64, 4), ([500, 77], [16, 5], 8, 2, 128, 16),
    ([300, 64, 200], [64, 64, 0], 8, 2, 128, 32), ([200, 700], [128, 100], 4, 2, 80, 24), ([140], [128], 3, 1, 100, 7),
    ([333, 90], [33, 31], 1, 1, 300, 16)])
def test_tree(dev, lens, news, h, hkv, d, page, window, sinks):
    rng = np.random.default_rng(sum(lens) + window)
    for deep in (False, True):
        print(f"tree lens={lens} news={news} h={h} hkv={hkv} d={d} window={window} sinks={sinks} deep={deep}", flush=True)
        Case(dev, lens, news, h, hkv, d, page, window, sinks, parents=[_tree(rng, n, deep) for n in news]).check()


def test_a_chain_as_a_tree_is_causal(dev):
    lens, news = [100, 260], [30, 128]
    chain = [[j - 1 for j in range(n)] for n in news]
    for window, sinks in ((0, 0), (25, 3)):
        a = Case(dev, lens, news, 4, 2, 64, 16, window, sinks)
        b = Case(dev, lens, news, 4, 2, 64, 16, window, sinks, parents=chain)
        compare(a.check(), b.check().astype(np.float64), tolerance(a.q, a.pool.k, a.pool.v, a.scale, 260))


def test_parents_that_are_not_below_are_roots(dev):
    c = Case(dev, [60], [6], 2, 2, 64, 16, parents=[[-1, 0, 5, 3, -9, 2**31 - 1]])
    c.check()  # the plain form treats them so


def test_a_whole_tree_before_the_first_key(dev):
    got = Case(dev, [3, 0], [7, 4], 4, 2, 64, 16, parents=[[-1, 0, 1, 2, 3, 4, 5], [-1, -1, 0, 1]]).check()
    assert np.all(got[:4] == 0) and np.all(got[7:] == 0)


def test_too_many_drafts_are_refused(dev):
    c = Case(dev, [200], [129], 2, 2, 64, 16, parents=[[-1] * 129])
    with pytest.raises(UnsupportedOperation):
        dev.check(c.call(dev._lib, dev.ctx), "attention")


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_drafts_of_other_branches_do_not_reach_a_row(dev, bad):
    parents = [[-1, 0, 1, -1, 3, 4, 0, 6], [-1] * 40]
    c = Case(dev, [100, 50], [8, 40], 4, 2, 64, 16, parents=parents)
    for b, j in ((0, 95), (0, 97), (1, 10 + 17), (1, 10 + 33)):
        c.pool.v[c.pool.table[b, j // 16], :, j % 16] = bad
        c.pool.k[c.pool.table[b, j // 16], 0, j % 16] = bad
    c.upload()
    c.check()


# ---- dense operands ----------------------------------------------------------------------------------


@pytest.mark.parametrize("b,h,hkv,sq,skv,d,window,sinks", [
    (1, 1, 1, 1, 1, 64, 0, 0), (2, 4, 2, 70, 70, 64, 16, 2), (1, 8, 8, 257, 257, 128, 100, 4), (2, 6, 3, 33, 400, 80, 64, 0),
    (1, 4, 1, 1, 1000, 128, 300, 4), (3, 2, 2, 9, 5, 32, 3, 1), (1, 3, 3, 300, 300, 256, 50, 1), (1, 2, 2, 130, 130, 64, 1, 0),
    (1, 2, 1, 40, 41, 300, 10, 2), (1, 4, 4, 520, 520, 96, 0, 0)])
def test_dense(dev, b, h, hkv, sq, skv, d, window, sinks):
    rng = np.random.default_rng(sq + skv + d)
    q = rng.standard_normal((b, h, sq, d), dtype=np.float32)
    k, v = (rng.standard_normal((b, hkv, skv, d), dtype=np.float32) for _ in range(2))
    t = [Tensor.from_data(x, list(x.shape), dev) for x in (q, k, v)]
    got = t[0].sliding_window_attention(t[1], t[2], window, sinks).to_numpy().reshape(q.shape)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    see = visible(skv - sq, sq, window, sinks)
    tol = tolerance(q, k, v, scale, skv)
    for i in range(b):
        want = attend(q[i].transpose(1, 0, 2), k[i].transpose(1, 0, 2), v[i].transpose(1, 0, 2), see, scale)
        compare(got[i].transpose(1, 0, 2), want, tol)
    if window == 0 and h == hkv and sq == skv:  # the causal op's own result, to rounding
        c = t[0].causal_attention(t[1], t[2]).to_numpy().reshape(q.shape)
        assert np.abs(got - c).max() <= 2 * tol


def test_dense_windows_beyond_any_position(dev):
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((1, 2, 50, 64), dtype=np.float32) for _ in range(3))
    t = [Tensor.from_data(x, list(x.shape), dev) for x in (q, k, v)]
    want = t[0].sliding_window_attention(t[1], t[2], 0).to_numpy()
    for window, sinks in ((50, 0), (2**31 - 1, 2**31 - 1), (2**40, 0), (1, 50), (3, 2**40)):
        assert np.array_equal(t[0].sliding_window_attention(t[1], t[2], window, sinks).to_numpy(), want), (window, sinks)


@pytest.mark.parametrize("sq,skv", [(300, 100), (20, 7), (129, 128)])
def test_dense_windows_beyond_any_position_with_more_rows_than_keys(dev, sq, skv):
    rng = np.random.default_rng(sq)
    q = rng.standard_normal((1, 2, sq, 64), dtype=np.float32)
    k, v = (rng.standard_normal((1, 2, skv, 64), dtype=np.float32) for _ in range(2))
    t = [Tensor.from_data(x, list(x.shape), dev) for x in (q, k, v)]
    want = t[0].sliding_window_attention(t[1], t[2], 0).to_numpy()
    for window in (skv, 2**31 - 1, 2**31 - 200):
        assert np.array_equal(t[0].sliding_window_attention(t[1], t[2], window).to_numpy(), want), window


def test_dense_strides_and_empty_batches(dev):
    """[B, S, H, D] operands with padding between the rows, as a projection writes them."""
    b, h, hkv, sq, skv, d, pad = 2, 4, 2, 60, 75, 64, 5
    rng = np.random.default_rng(5)
    def put(heads, s):
        x = np.full((b, s, heads * d + pad), np.nan, np.float32)
        x[..., :heads * d] = rng.standard_normal((b, s, heads * d), dtype=np.float32)
        return (x[..., :heads * d].reshape(b, s, heads, d), Tensor.from_data(x, [x.size], dev),
                N.AttnLayout(s * (heads * d + pad), d, heads * d + pad))
    (q, tq, lq), (k, tk, lk), (v, tv, lv) = put(h, sq), put(hkv, skv), put(hkv, skv)
    to, lo = Tensor.from_data(np.full((b, sq, h * d + pad), 7.0), [b * sq * (h * d + pad)], dev), lq
    dev.check(dev._lib.bch_sdpa_window(dev.ctx, b, h, hkv, sq, skv, d, 0.125, 20, 3, C.c_void_p(tq.ptr), lq,
                                       C.c_void_p(tk.ptr), lk, C.c_void_p(tv.ptr), lv, C.c_void_p(to.ptr), lo), "window")
    out = to.to_numpy().reshape(b, sq, h * d + pad)
    assert np.all(out[..., h * d:] == 7.0)
    for i in range(b):
        want = attend(q[i], k[i], v[i], visible(skv - sq, sq, 20, 3), 0.125)
        compare(out[i, :, :h * d].reshape(sq, h, d), want, tolerance(q, k, v, 0.125, skv))
    e = Tensor.empty([0, 2, 5, 8], dev)
    assert e.sliding_window_attention(e, e, 3).shape() == [0, 2, 5, 8]


# ---- offsets beyond 32 bits, graphs, streams ------------------------------------------------------------


def test_offsets_beyond_32_bits(dev):
    """Pages 2^29 floats apart: the fifth and later ones lie beyond 2^31 floats."""
    c = Case(dev, [100, 45], [1, 40], 4, 2, 64, 16, 60, 2)
    apart, num = 1 << 29, 12
    assert c.pool.num >= num
    big = [Tensor.empty([(num - 1) * apart + 2 * 16 * 64], dev) for _ in range(2)]
    table = np.full_like(c.pool.table, -1)
    for at, (i, j) in enumerate(np.argwhere(c.pool.table >= 0)[:num]):
        p = num - 1 - at
        table[i, j] = p
        for t, x in zip(big, (c.pool.k, c.pool.v)):
            dev.upload(t.ptr + 4 * p * apart, x[c.pool.table[i, j]])
    c.pool.table = np.where(table >= 0, c.pool.table, -1)  # what did not find a place is not held
    c.i32 = _I32(dev, c.start, c.lens, table)
    lay = N.AttnLayout(apart, 16 * 64, 64)
    c.kv = N.KvPages(big[0].ptr, big[1].ptr, lay, lay, num, 16, 2, 64, c.i32.ptrs[2], table.shape[1])
    c.batch.start, c.batch.len = c.i32.ptrs[0], c.i32.ptrs[1]
    c.check()


@pytest.mark.parametrize("lens,news,tree", [([700, 30], [1, 1], False), ([2000, 90], [90, 33], False), ([900, 200], [20, 64], True)])
def test_captured_calls_read_lengths_at_replay(dev, lens, news, tree):
    """A graph replayed with other lengths and pages in the same buffers gives the other result; eager calls and
    a larger workspace in between do not disturb it."""
    hip = _hip()
    rng = np.random.default_rng(1)
    parents = [_tree(rng, n, True) for n in news] if tree else None
    a = Case(dev, lens, news, 8, 2, 128, 16, 300, 4, parents=parents)
    with _FreshCtx(dev) as f:
        graph, exe = C.c_void_p(), C.c_void_p()
        for warm in (False, True):  # first without a workspace, then with one
            if warm:
                assert a.call(f.lib, f.ctx) == N.BCH_OK and f.lib.bch_sync(f.ctx) == N.BCH_OK
            assert hip.hipStreamBeginCapture(f.stream, CAPTURE_RELAXED) == 0
            st = a.call(f.lib, f.ctx)
            assert hip.hipStreamEndCapture(f.stream, C.byref(graph)) == 0
            assert st == N.BCH_OK
            try:
                assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
                for shift in (0, 3, 17, 0):
                    shorter = [max(n, length - shift) for length, n in zip(lens, news)]
                    dev.upload(a.i32.ptrs[1], np.array(shorter, np.int32))
                    dev.upload(a.to.ptr, np.full(a.to.len(), 7.0, np.float32))
                    assert hip.hipGraphLaunch(exe, f.stream) == 0 and f.lib.bch_sync(f.ctx) == N.BCH_OK
                    a.lens = shorter
                    got = a.output()
                    compare(got, a.want(), tolerance(a.q, a.pool.k, a.pool.v, a.scale, max(lens)))
                    assert a.call(f.lib, f.ctx) == N.BCH_OK and f.lib.bch_sync(f.ctx) == N.BCH_OK
                    compare(a.output(), a.want(), tolerance(a.q, a.pool.k, a.pool.v, a.scale, max(lens)))
                    if shift == 3:
                        assert f.lib.bch_ctx_reserve(f.ctx, f.ws_bytes() + (1 << 22)) == N.BCH_OK
            finally:
                hip.hipGraphExecDestroy(exe)
                hip.hipGraphDestroy(graph)
            a.lens = list(lens)
            dev.upload(a.i32.ptrs[1], np.array(lens, np.int32))


def test_two_contexts_at_once(dev):
    """Two calls in flight on two contexts' streams, each with its own workspace."""
    a = Case(dev, [3000, 40], [1, 1], 8, 2, 128, 16, seed=1)
    b = Case(dev, [2500, 90], [2, 3], 8, 2, 128, 16, seed=2)
    with _FreshCtx(dev) as f, _FreshCtx(dev) as g:
        for _ in range(5):
            assert a.call(f.lib, f.ctx) == N.BCH_OK
            assert b.call(g.lib, g.ctx) == N.BCH_OK
        assert f.lib.bch_sync(f.ctx) == N.BCH_OK and g.lib.bch_sync(g.ctx) == N.BCH_OK
    for c in (a, b):
        compare(c.output(), c.want(), tolerance(c.q, c.pool.k, c.pool.v, c.scale, max(c.lens)))
