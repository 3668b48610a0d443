"""Where KvCache.append_rotary puts new tokens, without a GPU: one behind the last key that the sequence holds, whatever keep,
retain, truncate and fork have made of it.  The device is a stand-in whose calls note the positions that they turn by."""
from __future__ import annotations

import numpy as np
import pytest

from barracuda_amd import KvCache, Rotary, Tensor
from barracuda_amd import _native as N
from barracuda_amd.error import InvalidInput, InvalidOperation, OutOfMemory
from tests.rotary_model import depths
from tests.test_kv_cache_host import _HostDevice, _HostLib, _check_pages

HKV, D, H = 2, 4, 3


class _TurningLib(_HostLib):
    """A turn writes the position into the row's first column, and copies the others."""

    def bch_rotary(self, ctx, b, h, s, d, plan, inverse, first, positions, x, xl, o, ol):
        self.calls.append("rotary")
        assert b == 1 and (xl.head_stride, xl.row_stride) == (ol.head_stride, ol.row_stride) == (d, h * d)
        src, dst = (self._floats(p.value, s * h * d).reshape(s, h, d) for p in (x, o))
        dst[:] = src
        dst[:, :, 0] = self._ints(positions, s)[:, None]
        return N.BCH_OK

    def bch_kv_append_rotary(self, ctx, kv, batch, parent, plan, h, q, ql, o, ol, k, kl, v, vl):
        start, lens = self._ints(batch.start, batch.B + 1), self._ints(batch.len, batch.B)
        where = np.empty(batch.total)
        for b in range(batch.B):
            n = start[b + 1] - start[b]
            tree = self._ints(parent, batch.total)[start[b]:start[b + 1]] if parent is not None else range(-1, n - 1)
            where[start[b]:start[b + 1]] = lens[b] - n + np.array(depths(tree))
        kept = self._floats(k.value, batch.total * kv.Hkv * kv.D).reshape(-1, kv.Hkv, kv.D)
        turned = kept.copy()
        turned[:, :, 0] = where[:, None]
        for src, dst, heads in ((q, o, h),):
            a, b = (self._floats(p.value, batch.total * heads * kv.D).reshape(-1, heads, kv.D) for p in (src, dst))
            b[:] = a
            b[:, :, 0] = where[:, None]
        before = kept.copy()
        kept[:] = turned
        self.bch_kv_append(ctx, kv, batch, k, kl, v, vl)
        self.calls[-1] = "append_rotary"
        kept[:] = before
        return N.BCH_OK


def _device():
    dev = _HostDevice()
    dev._lib = _TurningLib()
    return dev


def _turn(cache, step, rotary):
    """append_rotary in every layer; the position of each new token, at which q and k and all layers agree."""
    x = lambda h: Tensor.from_data(np.full((step.total, h, D), 7.0), [step.total, h, D], cache.device)
    out = None
    for layer in range(cache.layers):
        q, k, v = x(H), x(HKV), x(HKV)
        got = cache.append_rotary(step, layer, rotary, q, k, v).to_numpy()
        assert np.all(got[:, :, 0] == got[:, :1, 0]) and np.all(got[:, :, 1:] == 7.0)
        assert np.all(q.to_numpy() == 7.0) and np.all(k.to_numpy() == 7.0)
        assert out is None or np.array_equal(out, got[:, 0, 0])
        out = got[:, 0, 0]
    return out.astype(int).tolist()


def _keys(cache, seq):
    """The positions that the sequence's keys were turned by; None where the page is gone."""
    k, v = cache.k.to_numpy(), cache.v.to_numpy()
    out = []
    for j in range(cache.length(seq)):
        p = cache.pages(seq)[j // cache.page_size]
        at = k[:, p, :, j % cache.page_size]
        assert p < 0 or (np.all(at[..., 0] == at[0, 0, 0]) and np.all(v[:, p, :, j % cache.page_size] == 7.0))
        out.append(int(at[0, 0, 0]) if p >= 0 else None)
    return out


def test_tokens_behind_retained_keys():
    dev = _device()
    cache, r = KvCache(2, 64, 4, HKV, D, dev), Rotary(D, device=dev)
    a = cache.new_sequence()
    assert _turn(cache, cache.batch([(a, 100)]), r) == list(range(100))
    cache.retain(a, [0, 1, 2, 3] + list(range(60, 100)))
    assert cache.length(a) == 44
    assert _turn(cache, cache.batch([(a, 2)]), r) == [100, 101]
    assert _keys(cache, a) == [0, 1, 2, 3] + list(range(60, 102))
    b = cache.fork(a)
    cache.retain(b, [0, 4, 5, 44])  # again, over the first gap
    cache.truncate(a, 20)           # behind key 75
    step = cache.batch([(b, 1), (a, 3)], parents=[[-1], [-1, 0, 0]])
    assert _turn(cache, step, r) == [101, 76, 77, 77]
    cache.keep(step, [[0], [0, 2]])
    assert _turn(cache, cache.batch([(a, 1), (b, 2)]), r) == [78, 102, 103]
    cache.truncate(a, 3)  # before the gap
    assert _turn(cache, cache.batch([(a, 2)]), r) == [3, 4]
    assert _keys(cache, a) == [0, 1, 2, 3, 4]


def test_drafts_kept_by_retain_and_lists_with_gaps():
    dev = _device()
    cache, r = KvCache(1, 64, 4, HKV, D, dev), Rotary(D, device=dev)
    a, b, c = (cache.new_sequence() for _ in range(3))
    tree = [-1, 0, 0, 2, -1]
    step = cache.batch([(a, 5), (b, 5), (c, 8)], parents=[tree, tree, list(range(-1, 7))])
    assert _turn(cache, step, r)[:5] == [0, 1, 1, 2, 0]
    # a branch is consecutive; a chain's tokens 0, 3 and 7 are not
    cache.keep(step, [[0, 2, 3], [0, 2, 3], [0, 3, 7]])
    assert _turn(cache, cache.batch([(a, 1), (b, 1), (c, 1)]), r) == [3, 3, 8]
    d = cache.new_sequence()
    assert _turn(cache, cache.batch([(d, 5)], parents=[tree]), r) == [0, 1, 1, 2, 0]
    cache.retain(d, [0, 2, 3])
    assert _turn(cache, cache.batch([(d, 1)]), r) == [3]
    cache.retain(d, [])
    assert _turn(cache, cache.batch([(d, 1)]), r) == [0]


@pytest.mark.parametrize("seed", range(12))
def test_random_programs(seed):
    """Against lists of every key's position."""
    rng = np.random.default_rng(seed)
    dev = _device()
    cache, r = KvCache(int(rng.integers(1, 3)), 40, int(rng.integers(1, 6)), HKV, D, dev), Rotary(D, device=dev)
    model = {}
    for _ in range(80):
        op = rng.choice(["batch", "batch", "drafts", "left", "new", "fork", "truncate", "free", "compact", "retain", "prefix"])
        seqs = list(model)
        if op == "new" or not seqs:
            model[cache.new_sequence()] = []
        elif op in ("batch", "drafts", "left"):
            chosen = [s for s in seqs if rng.random() < 0.7]
            counts = [int(rng.integers(0, 6)) for _ in chosen]
            parents = [[int(rng.integers(-1, j)) if j else -1 for j in range(n)] for n in counts]
            try:
                step = cache.batch(zip(chosen, counts), parents if op != "batch" else None)
            except OutOfMemory:
                continue
            got = _turn(cache, step, r)
            for i, (s, n) in enumerate(zip(chosen, counts)):
                first = model[s][-1] + 1 if model[s] else 0
                want = [first + x for x in (depths(parents[i]) if op != "batch" else range(n))]
                assert got[step.start[i]:step.start[i + 1]] == want
                model[s] = model[s] + want
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
            elif op in ("truncate", "prefix"):
                n = int(rng.integers(0, len(model[s]) + 1))
                cache.truncate(s, n) if op == "truncate" else cache.retain(s, range(n))
                model[s] = model[s][:n]
            elif op == "retain":
                ids = [j for j in range(len(model[s])) if rng.random() < 0.6]
                try:
                    cache.retain(s, ids)
                    model[s] = [model[s][j] for j in ids]
                except OutOfMemory:
                    pass
            elif op == "free":
                cache.free(s)
                del model[s]
            else:
                cache.compact()
        _check_pages(cache)
        for s, keys in model.items():
            assert _keys(cache, s) == keys, (op, s)


def test_sequences_as_they_were_appended_take_one_call():
    dev = _device()
    cache, r = KvCache(1, 64, 4, HKV, D, dev), Rotary(D, device=dev)
    a, b = cache.new_sequence(), cache.new_sequence()
    _turn(cache, cache.batch([(a, 9), (b, 3)]), r)
    cache.retain(a, range(7))
    cache.retain(b, [0, 2])
    dev._lib.calls.clear()
    _turn(cache, cache.batch([(a, 1), (b, 0)]), r)
    assert dev._lib.calls == ["append_rotary"]
    assert _turn(cache, cache.batch([(a, 1), (b, 1)]), r) == [8, 3]
    assert dev._lib.calls[1:] == ["rotary", "rotary", "append"]


def test_a_failed_batch_leaves_positions_as_they_were():
    dev = _device()
    cache, r = KvCache(1, 8, 4, HKV, D, dev), Rotary(D, device=dev)
    a = cache.new_sequence()
    _turn(cache, cache.batch([(a, 6)]), r)
    cache.retain(a, [0, 5])
    dev.fail_uploads = True
    with pytest.raises(OutOfMemory):
        cache.batch([(a, 3)], parents=[[-1, -1, 0]])
    dev.fail_uploads = False
    assert _turn(cache, cache.batch([(a, 1)]), r) == [6]


def test_positions_beyond_32_bits_are_refused():
    """A sequence that closes its keys up again and again stands ever further on; keys can still be appended as they are."""
    dev = _device()
    cache, r = KvCache(1, 8, 4, HKV, D, dev), Rotary(D, device=dev)
    a = cache.new_sequence()
    _turn(cache, cache.batch([(a, 2)]), r)
    cache._seqs[a].shifts = [(1, 2**31 - 3)]  # its last key at 2^31 - 2
    cache.append_rotary(cache.batch([(a, 1)]), 0, r, *(Tensor.from_data(np.zeros((1, h, D)), [1, h, D], dev) for h in (H, HKV, HKV)))
    cache.truncate(a, 2)
    step = cache.batch([(a, 2)])
    x = [Tensor.from_data(np.zeros((2, h, D)), [2, h, D], dev) for h in (H, HKV)]
    with pytest.raises(InvalidOperation):
        cache.append_rotary(step, 0, r, x[0], x[1], x[1])
    cache.append(step, 0, x[1], x[1])


def test_frequencies_beyond_what_angles_hold_are_refused():
    dev = _device()
    assert Rotary(4, freqs=[2.0**19, -(2.0**19)], device=dev).freqs[0] == 2.0**19
    for bad in ([1.0, 2.0**19 + 1], [-1e6, 0.0], [np.inf, 1.0], [1.0, np.nan]):
        with pytest.raises(InvalidInput):
            Rotary(4, freqs=bad, device=dev)
    with pytest.raises(InvalidInput):
        Rotary(64, base=1e-9, device=dev)
