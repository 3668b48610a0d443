"""KvCache's bookkeeping without a GPU: pages taken, shared, copied before they are written, given back and
compacted, against a model that keeps every sequence's keys as a list.  The device is a stand-in whose
memory is the host's and whose calls are the plain forms.  Also the C ABI's refusals, which come before any
device call."""
from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest

from barracuda_amd import _native as N
from barracuda_amd import KvCache, SlidingWindowAttention, Tensor
from barracuda_amd.error import InvalidInput, InvalidOperation, OutOfMemory, ShapeMismatch
from tests.kv_model import visible


class _HostLib:
    """The cache's calls over host memory."""

    def __init__(self):
        self.calls = []

    @staticmethod
    def _floats(ptr, n):
        return np.ctypeslib.as_array(C.cast(ptr, C.POINTER(C.c_float)), (n,))

    @staticmethod
    def _ints(ptr, n):
        ptr = ptr.value if isinstance(ptr, C.c_void_p) else ptr
        return np.ctypeslib.as_array(C.cast(ptr, C.POINTER(C.c_int)), (n,))

    def _pool(self, kv, which, layers=1, stride=0):
        page = kv.k_layout.batch_stride
        return self._floats(kv.k if which == "k" else kv.v, (layers - 1) * stride + kv.num_pages * page)

    def bch_kv_append(self, ctx, kv, batch, k, kl, v, vl):
        self.calls.append("append")
        start, lens = self._ints(batch.start, batch.B + 1), self._ints(batch.len, batch.B)
        table = self._ints(kv.table, batch.B * kv.table_width).reshape(batch.B, -1)
        for which, new in (("k", k), ("v", v)):
            pool = self._pool(kv, which).reshape(kv.num_pages, kv.Hkv, kv.page_size, kv.D)
            rows = self._floats(new.value, batch.total * kv.Hkv * kv.D).reshape(-1, kv.Hkv, kv.D)
            for b in range(batch.B):
                n = start[b + 1] - start[b]
                for i in range(n):
                    j = lens[b] - n + i
                    pool[table[b, j // kv.page_size], :, j % kv.page_size] = rows[start[b] + i]
        return N.BCH_OK

    def bch_kv_copy_pages(self, ctx, kv, layers, ks, vs, n, src, dst):
        self.calls.append(("copy", n))
        assert len(set(dst[:n])) == n and not set(dst[:n]) & set(src[:n])
        for which in "kv":
            pool = self._pool(kv, which, layers, ks).reshape(layers, kv.num_pages, -1)
            for x in range(n):
                pool[:, dst[x]] = pool[:, src[x]]
        return N.BCH_OK

    def bch_kv_keep(self, ctx, kv, layers, ks, vs, b, total, start, keep, to):
        self.calls.append("keep")
        start, keep, to = self._ints(start, b + 1), self._ints(keep, total), self._ints(to, b)
        table = self._ints(kv.table, b * kv.table_width).reshape(b, -1)
        ps = kv.page_size
        for which in "kv":
            pool = self._pool(kv, which, layers, ks).reshape(layers, kv.num_pages, kv.Hkv, ps, kv.D)
            for s in range(b):
                for i, j in enumerate(keep[start[s]:start[s + 1]]):
                    t = to[s] + i
                    assert j >= t
                    pool[:, table[s, t // ps], :, t % ps] = pool[:, table[s, j // ps], :, j % ps]
        return N.BCH_OK


class _HostDevice:
    """What Tensor and KvCache ask of a device."""

    def __init__(self):
        self._lib, self._lock, self.ctx, self.mem = _HostLib(), threading.RLock(), None, {}
        self.fail_uploads = False

    def name(self):
        return "host"

    def check(self, status, op):
        assert status == N.BCH_OK

    def alloc(self, nbytes):
        a = np.full(nbytes, 0xff, np.uint8)  # NaN as floats
        self.mem[a.ctypes.data] = a
        return a.ctypes.data

    def free(self, ptr):
        self.mem.pop(ptr, None)

    def upload(self, ptr, host):
        if self.fail_uploads:
            raise OutOfMemory("planted")
        host = np.ascontiguousarray(host)
        C.memmove(ptr, host.ctypes.data, host.nbytes)

    def download(self, ptr, nbytes):
        return np.frombuffer(C.string_at(ptr, nbytes), np.float32).copy()


def _cache(layers=2, pages=24, page=4, heads=2, d=3):
    return KvCache(layers, pages, page, heads, d, _HostDevice())


def _append(cache, step, serial):
    """Append numbered keys to every layer: key number s is s + layer / 8 in all its elements, value its negative."""
    numbers = np.arange(serial, serial + step.total)
    for layer in range(cache.layers):
        x = np.broadcast_to((numbers + layer / 8.0)[:, None, None], (step.total, cache.kv_heads, cache.head_dim))
        x = x.astype(np.float32)
        shape = list(x.shape)
        cache.append(step, layer, Tensor.from_data(x, shape, cache.device), Tensor.from_data(-x, shape, cache.device))
    return numbers


def _read(cache, seq):
    """The numbers of a sequence's keys, None where the page is gone; all layers, heads and K against V agree."""
    k = cache.k.to_numpy()
    v = cache.v.to_numpy()
    out = []
    for j in range(cache.length(seq)):
        p = cache.pages(seq)[j // cache.page_size]
        if p < 0:
            out.append(None)
            continue
        at = k[:, p, :, j % cache.page_size]
        for layer in range(cache.layers):
            assert np.all(at[layer] == at[0, 0, 0] + layer / 8.0)
        assert np.array_equal(at, -v[:, p, :, j % cache.page_size])
        out.append(int(at[0, 0, 0]))
    return out


def _check_pages(cache):
    held = {}
    for s in cache._seqs.values():
        for p in s.pages:
            if p >= 0:
                held[p] = held.get(p, 0) + 1
    assert [held.get(p, 0) for p in range(cache.num_pages)] == cache._refs
    assert sorted(cache._free) == [p for p in range(cache.num_pages) if p not in held]


@pytest.mark.parametrize("seed", range(12))
def test_random_programs_keep_every_sequence(seed):
    """Random appends, forks, keeps, evictions, truncations, frees and compactions against lists of numbers."""
    rng = np.random.default_rng(seed)
    cache = _cache(page=int(rng.integers(1, 6)), pages=30)
    model, serial = {}, 0
    for _ in range(60):
        op = rng.choice(["batch", "batch", "drafts", "new", "fork", "evict", "truncate", "free", "compact", "retain"])
        seqs = list(model)
        if op == "new" or not seqs:
            model[cache.new_sequence()] = []
        elif op in ("batch", "drafts"):
            chosen = [s for s in seqs if rng.random() < 0.7]
            counts = [int(rng.integers(0, 6)) for _ in chosen]
            parents = [[int(rng.integers(-1, j)) if j else -1 for j in range(n)] for n in counts]
            before = {s: (cache.pages(s), cache.length(s)) for s in seqs}
            try:
                step = cache.batch(zip(chosen, counts), parents if op == "drafts" else None)
            except (OutOfMemory, InvalidOperation):
                assert before == {s: (cache.pages(s), cache.length(s)) for s in seqs}
                continue
            numbers = _append(cache, step, serial)
            serial += step.total
            for i, s in enumerate(chosen):
                model[s] = model[s] + list(numbers[step.start[i]:step.start[i + 1]])
            if op == "drafts":
                kept = [[j for j in range(n) if rng.random() < 0.5] for n in counts]
                cache.keep(step, kept)
                for s, n, ids in zip(chosen, counts, kept):
                    old = len(model[s]) - n
                    model[s] = model[s][:old] + [model[s][old + x] for x in ids]
        else:
            s = seqs[int(rng.integers(len(seqs)))]
            if op == "fork":
                model[cache.fork(s)] = list(model[s])
            elif op == "evict":
                window, sinks = int(rng.integers(1, 9)), int(rng.integers(0, 3))
                cache.evict(s, window, sinks)
                for j, x in enumerate(_read(cache, s)):
                    if x is None and model[s][j] is not None:  # given back just now
                        assert sinks <= j <= len(model[s]) - window
                        model[s][j] = None
            elif op == "truncate":
                n = int(rng.integers(0, len(model[s]) + 1))
                cache.truncate(s, n)
                model[s] = model[s][:n]
            elif op == "retain":
                ids = [j for j in range(len(model[s])) if rng.random() < 0.6]
                try:
                    cache.retain(s, ids)
                    model[s] = [model[s][j] for j in ids]
                except (InvalidOperation, OutOfMemory):
                    pass
            elif op == "free":
                cache.free(s)
                del model[s]
            else:
                cache.compact()
                live = cache.num_pages - cache.free_pages()
                assert all(p < live for t in model for p in cache.pages(t))
        _check_pages(cache)
        for s, keys in model.items():
            assert _read(cache, s) == keys, (op, s)


def test_a_shared_page_is_copied_once_per_writer_but_the_last():
    cache = _cache(page=4)
    a = cache.new_sequence()
    _append(cache, cache.batch([(a, 6)]), 0)
    b, c = cache.fork(a), cache.fork(a)
    cache.device._lib.calls.clear()
    step = cache.batch([(a, 1), (b, 1), (c, 1)])
    assert cache.device._lib.calls == [("copy", 2)]
    _append(cache, step, 100)
    assert [_read(cache, s)[4:] for s in (a, b, c)] == [[4, 5, 100], [4, 5, 101], [4, 5, 102]]
    assert cache.pages(a)[0] == cache.pages(b)[0] == cache.pages(c)[0]
    _check_pages(cache)


def test_out_of_pages_changes_nothing():
    cache = _cache(pages=4, page=4)
    a = cache.new_sequence()
    _append(cache, cache.batch([(a, 15)]), 0)
    b = cache.fork(a)
    with pytest.raises(OutOfMemory):
        cache.batch([(b, 1)])
    assert cache.length(b) == 15 and cache.pages(b) == cache.pages(a) and cache.free_pages() == 0
    cache.free(a)
    _append(cache, cache.batch([(b, 1)]), 50)
    assert _read(cache, b) == list(range(15)) + [50]
    with pytest.raises(OutOfMemory):
        cache.batch([(b, 1)])


def test_a_failed_upload_leaves_the_sequences_as_they_were():
    cache = _cache()
    a = cache.new_sequence()
    _append(cache, cache.batch([(a, 5)]), 0)
    cache.device.fail_uploads = True
    with pytest.raises(OutOfMemory):
        cache.batch([(a, 9)])
    cache.device.fail_uploads = False
    assert cache.length(a) == 5
    _check_pages(cache)
    _append(cache, cache.batch([(a, 9)]), 5)
    assert _read(cache, a) == list(range(14))


def test_stale_steps_and_bad_arguments_are_refused():
    cache = _cache()
    a = cache.new_sequence()
    step = cache.batch([(a, 3)])
    x = Tensor.from_data(np.zeros((3, 2, 3)), [3, 2, 3], cache.device)
    cache.append(step, 0, x, x)
    with pytest.raises(InvalidInput):
        cache.append(step, 2, x, x)
    with pytest.raises(ShapeMismatch):
        cache.append(step, 0, x, Tensor.from_data(np.zeros((2, 2, 3)), [2, 2, 3], cache.device))
    with pytest.raises(InvalidInput):
        cache.batch([(a, 1), (a, 1)])
    with pytest.raises(InvalidInput):
        cache.batch([(a, -1)])
    with pytest.raises(InvalidInput):
        cache.batch([(99, 1)])
    for parents in ([[0]], [[-2]], [[-1, -1]], [], [[-1], [-1]]):
        with pytest.raises(InvalidInput):
            cache.batch([(a, 1)], parents)
    with pytest.raises(InvalidInput):
        cache.batch([(a, 129)], [[-1] * 129])
    for kept in ([[1, 0]], [[3]], [[0, 0]], [[-1]], [[0], [0]]):
        with pytest.raises(InvalidInput):
            cache.keep(step, kept)
    with pytest.raises(InvalidInput):
        cache.attention(step, 0, Tensor.from_data(np.zeros((3, 3, 3)), [3, 3, 3], cache.device))
    with pytest.raises(ShapeMismatch):
        cache.attention(step, 0, Tensor.from_data(np.zeros((3, 2, 4)), [3, 2, 4], cache.device))
    with pytest.raises(InvalidInput):
        cache.attention(step, 0, x, window=-1)
    with pytest.raises(InvalidInput):
        cache.evict(a, 0)
    with pytest.raises(InvalidInput):
        cache.truncate(a, 4)
    with pytest.raises(InvalidInput):
        cache.retain(a, [1, 1])
    other = KvCache(2, 24, 4, 2, 3, cache.device)
    with pytest.raises(InvalidInput):
        other.append(step, 0, x, x)
    cache.truncate(a, 2)
    with pytest.raises(InvalidOperation):
        cache.append(step, 0, x, x)
    with pytest.raises(InvalidOperation):
        cache.keep(step, [[0]])
    with pytest.raises(InvalidInput):
        KvCache(1, 0, 4, 2, 3, cache.device)


def test_keep_of_a_step_with_a_later_one_behind_is_refused():
    cache = _cache()
    a = cache.new_sequence()
    first = cache.batch([(a, 3)])
    _append(cache, first, 0)
    _append(cache, cache.batch([(a, 1)]), 3)
    with pytest.raises(InvalidOperation):
        cache.keep(first, [[0]])
    assert _read(cache, a) == [0, 1, 2, 3]


def test_sliding_window_attention_checks_shapes():
    def t(*s):
        x = Tensor.__new__(Tensor)
        x._shape, x._device = list(s), None
        return x
    q, k = t(1, 4, 5, 8), t(1, 2, 9, 8)
    SlidingWindowAttention(q, k, k, 3, 1)
    with pytest.raises(InvalidInput):
        SlidingWindowAttention(t(1, 3, 5, 8), k, k, 3)
    with pytest.raises(InvalidInput):
        SlidingWindowAttention(q, k, k, -1)
    with pytest.raises(InvalidInput):
        SlidingWindowAttention(q, k, k, 1, -1)
    with pytest.raises(InvalidInput):
        SlidingWindowAttention(t(4, 5, 8), k, k, 3)
    with pytest.raises(ShapeMismatch):
        SlidingWindowAttention(q, k, t(1, 2, 8, 8), 3)
    with pytest.raises(ShapeMismatch):
        SlidingWindowAttention(q, t(2, 2, 9, 8), t(2, 2, 9, 8), 3)


def _pages(**over):
    lay = N.AttnLayout(64, 32, 8)
    kv = dict(k=16, v=16, k_layout=lay, v_layout=lay, num_pages=4, page_size=4, Hkv=2, D=8, table=16, table_width=2)
    kv.update(over)
    return N.KvPages(*[kv[f] for f, _ in N.KvPages._fields_])


def _batch(**over):
    b = dict(B=1, total=3, max_new=3, max_len=5, start=16, len=16)
    b.update(over)
    return N.KvBatch(*[b[f] for f, _ in N.KvBatch._fields_])


def test_c_calls_refuse_before_any_device_call():
    """No pointer here is ever followed: a call without a context gets no further than its checks."""
    lib, nul, x = N.load(), C.c_void_p(), C.c_void_p(16)
    row, thin = N.AttnLayout(0, 8, 16), N.AttnLayout(0, 8, 7)

    def attend(kv=None, batch=None, h=4, window=0, sinks=0, parent=None, ql=row, ol=row):
        return lib.bch_sdpa_paged(nul, kv or _pages(), batch or _batch(), h, 1.0, window, sinks, parent, x, ql, x, ol)

    E, S, U = N.BCH_E_INVALID, N.BCH_E_SHAPE, N.BCH_E_UNSUPPORTED
    assert attend() == E and "ctx is NULL" in N.last_error(None)
    assert lib.bch_sdpa_paged(nul, None, _batch(), 4, 1.0, 0, 0, None, x, row, x, row) == E
    assert lib.bch_sdpa_paged(nul, _pages(), None, 4, 1.0, 0, 0, None, x, row, x, row) == E
    for f in ("num_pages", "page_size", "Hkv", "D", "table_width"):
        assert attend(_pages(**{f: 0})) == S, f
    for f in ("k_layout", "v_layout"):
        assert attend(_pages(**{f: thin})) == E and "layout" in N.last_error(None)
        assert attend(_pages(**{f: N.AttnLayout(-1, 8, 8)})) == E
    for f in ("B", "total", "max_new", "max_len"):
        assert attend(batch=_batch(**{f: -1})) == S, f
    assert attend(h=0) == S
    assert attend(h=3) == E and "divisible" in N.last_error(None)
    assert attend(window=-1) == E and attend(sinks=-1) == E
    assert attend(ql=thin) == E and attend(ol=thin) == E
    wide = N.AttnLayout(4096, 2048, 2048)
    assert attend(_pages(D=1025, k_layout=wide, v_layout=wide), ql=wide, ol=wide) == U
    assert attend(batch=_batch(total=200, max_new=129), parent=x) == U and "drafts" in N.last_error(None)
    assert attend(batch=_batch(total=128, max_new=500), parent=x) == E  # at most `total` of them: only ctx is missing

    def dense(b=1, h=4, hkv=2, sq=3, skv=5, d=8, window=0, sinks=0, lay=row):
        return lib.bch_sdpa_window(nul, b, h, hkv, sq, skv, d, 1.0, window, sinks, x, lay, x, lay, x, lay, x, lay)
    assert dense() == E and "ctx is NULL" in N.last_error(None)
    for f in ("b", "h", "hkv", "sq", "skv", "d"):
        assert dense(**{f: 0}) == S, f
    assert dense(h=3) == E and dense(window=-1) == E and dense(sinks=-1) == E and dense(lay=thin) == E
    assert dense(d=1025, lay=wide) == U

    def append(kv=None, batch=None, kl=row, vl=row):
        return lib.bch_kv_append(nul, kv or _pages(), batch or _batch(), x, kl, x, vl)
    assert append() == E and "ctx is NULL" in N.last_error(None)
    assert append(_pages(page_size=0)) == S and append(batch=_batch(total=-1)) == S
    assert append(kl=thin) == E and append(vl=thin) == E

    def copy(src, dst, kv=None, layers=1, stride=0):
        arr = C.c_int * max(1, len(src))
        return lib.bch_kv_copy_pages(nul, kv or _pages(), layers, stride, stride, len(src), arr(*src), arr(*dst))
    assert copy([0], [1]) == E and "ctx is NULL" in N.last_error(None)
    assert copy([4], [1]) == E and "outside" in N.last_error(None)
    assert copy([0], [-1]) == E and copy([-1], [0]) == E and copy([0], [4]) == E
    assert copy([0, 0], [1, 1]) == E and "two copies" in N.last_error(None)
    assert copy([0, 1], [1, 2]) == E and "read and written" in N.last_error(None)
    assert copy([0], [0]) == E
    assert copy([0], [1], layers=-1) == S and copy([0], [1], stride=-1) == S
    assert lib.bch_kv_copy_pages(nul, _pages(), 1, 0, 0, -1, None, None) == S
    assert lib.bch_kv_copy_pages(nul, _pages(), 1, 0, 0, 1, None, None) == E

    def keep(b=1, total=3, kv=None, layers=1, stride=0):
        return lib.bch_kv_keep(nul, kv or _pages(), layers, stride, stride, b, total, x, x, x)
    assert keep() == E and "ctx is NULL" in N.last_error(None)
    assert keep(b=-1) == S and keep(total=-1) == S and keep(layers=-1) == S and keep(stride=-1) == S
    assert keep(b=65536) == U and keep(layers=32768) == U
    assert keep(kv=_pages(table_width=0)) == S


class _LimitedLib(_HostLib):
    """Refuses what bch_kv_keep refuses."""

    def bch_kv_keep(self, ctx, kv, layers, ks, vs, b, total, start, keep, to):
        if b > 65535 or layers > 32767:
            return N.BCH_E_UNSUPPORTED
        return super().bch_kv_keep(ctx, kv, layers, ks, vs, b, total, start, keep, to)


def test_keep_of_more_sequences_than_one_call_takes():
    """As many as one step may have; the ones with nothing to move among them."""
    cache = _cache(layers=1, pages=140000, page=1, heads=1, d=1)
    cache.device._lib = _LimitedLib()
    seqs = [cache.new_sequence() for _ in range(70000)]
    step = cache.batch([(s, 2) for s in seqs])
    _append(cache, step, 0)
    kept = [[] if s % 50 == 7 else [s % 3 // 2] for s in seqs]
    cache.keep(step, kept)
    k = cache.k.to_numpy().reshape(-1)
    for s, ids in zip(seqs, kept):
        assert [k[p] for p in cache.pages(s)] == [2 * s + x for x in ids]
    assert cache.device._lib.calls.count("keep") == 2


def test_keep_in_more_layers_than_one_call_takes():
    cache = _cache(layers=40000, pages=3, page=1, heads=1, d=1)
    cache.device._lib = _LimitedLib()
    a = cache.new_sequence()
    step = cache.batch([(a, 2)])
    old, new = cache.pages(a)
    for pool in (cache.k, cache.v):
        x = np.ctypeslib.as_array(C.cast(pool.ptr, C.POINTER(C.c_float)), (cache.layers, 3))
        x[:, new] = np.arange(cache.layers)
    cache.keep(step, [[1]])
    for pool in (cache.k, cache.v):
        assert np.array_equal(pool.to_numpy().reshape(-1, 3)[:, old], np.arange(cache.layers))


def test_a_failed_upload_leaves_a_step_that_can_be_kept():
    cache = _cache()
    a = cache.new_sequence()
    step = cache.batch([(a, 5)], [[-1, 0, 0, 1, 1]])
    _append(cache, step, 0)
    cache.device.fail_uploads = True
    with pytest.raises(OutOfMemory):
        cache.keep(step, [[0, 2, 4]])
    cache.device.fail_uploads = False
    assert cache.length(a) == 5
    cache.keep(step, [[0, 2, 4]])
    assert _read(cache, a) == [0, 2, 4]
    _check_pages(cache)


class _SeenLib(_HostLib):
    """Attention that only notes that it was called."""

    def bch_sdpa_paged(self, ctx, kv, batch, h, scale, window, sinks, parent, q, ql, o, ol):
        self.calls.append(("attention", window, sinks))
        return N.BCH_OK


def _attends(cache, step, window, sinks):
    """Whether attention through this window takes the step, and that it does in every layer or in none."""
    q = Tensor.from_data(np.zeros((step.total, 2, 3)), [step.total, 2, 3], cache.device)
    took = []
    for layer in range(cache.layers):
        n = len(cache.device._lib.calls)
        try:
            cache.attention(step, layer, q, window, sinks)
            took.append(True)
        except InvalidOperation as e:
            assert "evict" in str(e)
            took.append(False)
        assert (len(cache.device._lib.calls) > n) == (took[-1] and step.total > 0)
    assert len(set(took)) == 1
    return took[0]


def test_attention_that_would_see_evicted_keys_is_refused():
    """Evicted keys may not silently count as nothing: after a truncation, through a larger window or with more
    sinks than evict was told of, a row would see them."""
    cache = _cache(page=4)
    cache.device._lib = _SeenLib()
    a, b = cache.new_sequence(), cache.new_sequence()
    _append(cache, cache.batch([(a, 21), (b, 9)]), 0)
    assert cache.evict(a, window=8, sinks=3) == 2  # pages 1 and 2: keys 4 .. 11; the next token sees 14 on
    step = cache.batch([(a, 1), (b, 2)])
    assert _attends(cache, step, 8, 3) and _attends(cache, step, 10, 4) and _attends(cache, step, 1, 0)
    for window, sinks in ((0, 0), (11, 0), (2**40, 0), (8, 5), (8, 2**40)):
        assert not _attends(cache, step, window, sinks), (window, sinks)
    assert _attends(cache, cache.batch([(a, 0), (b, 1)]), 0, 0)  # no row of the sequence
    f = cache.fork(a)
    cache.truncate(a, 17)
    step = cache.batch([(a, 2), (f, 2)], [[-1, 0], [-1, -1]])  # now key 17 would see 10 and 11 through 8
    assert not _attends(cache, step, 8, 3) and _attends(cache, step, 6, 3)
    assert _attends(cache, cache.batch([(f, 1)]), 8, 3)
    cache.retain(a, [0, 1, 2, 3])
    step = cache.batch([(a, 1)])
    assert _attends(cache, step, 0, 0)


@pytest.mark.parametrize("seed", range(6))
def test_attention_is_refused_exactly_where_an_evicted_key_would_be_seen(seed):
    rng = np.random.default_rng(seed)
    cache = _cache(page=int(rng.integers(1, 5)), pages=60)
    cache.device._lib = _SeenLib()
    for _ in range(40):
        seqs = [cache.new_sequence() for _ in range(2)]
        _append(cache, cache.batch([(s, int(rng.integers(1, 30))) for s in seqs]), 0)
        for s in seqs:
            for _ in range(int(rng.integers(0, 3))):
                cache.evict(s, int(rng.integers(1, 12)), int(rng.integers(0, 6)))
            if rng.random() < 0.4:
                cache.truncate(s, int(rng.integers(0, cache.length(s) + 1)))
        counts = [int(rng.integers(0, 4)) for _ in seqs]
        parents = [[int(rng.integers(-1, j)) if j else -1 for j in range(n)] for n in counts] if rng.random() < 0.5 else None
        try:
            step = cache.batch(zip(seqs, counts), parents)
        except InvalidOperation:
            counts = [0, 0]
            step = cache.batch(zip(seqs, counts))
            parents = None
        window, sinks = int(rng.integers(0, 14)), int(rng.integers(0, 8))
        hidden = False
        for i, (s, n) in enumerate(zip(seqs, counts)):
            see = visible(cache.length(s) - n, n, window, sinks, parents[i] if parents else None).any(0)
            hidden |= any(x and cache.pages(s)[j // cache.page_size] < 0 for j, x in enumerate(see))
        assert _attends(cache, step, window, sinks) == (not hidden), (window, sinks)
        for s in seqs:
            cache.free(s)


def test_sequences_longer_than_the_kernels_count_are_refused():
    """2^31 - 256 keys: a longer length counts as that many, and its last tokens would go astray."""
    cache = _cache(page=1, pages=1, heads=1, d=1, layers=1)
    a = cache.new_sequence()
    cache._seqs[a].length = 2**31 - 256 - 2
    with pytest.raises(InvalidInput):
        cache.batch([(a, 3)])
    with pytest.raises(OutOfMemory):  # up to there only the pages are missing
        cache.batch([(a, 2)])
