"""Rotary positions without a GPU: the frequencies of the scalings, and the refusals, which come before any device call."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from barracuda_amd import KvCache, Rotary, RotaryPositions, Tensor, rotary_freqs
from barracuda_amd import _native as N
from barracuda_amd.error import DeviceError, InvalidInput, InvalidOperation, ShapeMismatch
from tests.test_kv_cache_host import _HostDevice, _batch, _pages


def test_frequencies():
    f = rotary_freqs(8, base=10000.0)
    assert np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-15)
    assert np.allclose(rotary_freqs(8, scaling="linear", factor=4.0), f / 4, rtol=1e-15)
    g = rotary_freqs(8, scaling="base", factor=4.0)
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-14) and np.all(g[1:] < f[1:])
    assert np.array_equal(rotary_freqs(2, scaling="base", factor=4.0), [1.0])
    g = rotary_freqs(128, scaling="parts", factor=8.0, context=4096.0)
    turns = 4096.0 * rotary_freqs(128) / (2 * math.pi)
    f = rotary_freqs(128)
    assert np.array_equal(g[turns >= 32], f[turns >= 32]) and np.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and np.all((g[between] < f[between]) & (g[between] > f[between] / 8))
    assert np.all(np.diff(g) < 0)


@pytest.mark.parametrize("kwargs", [{"dim": 3}, {"dim": 0}, {"dim": -2}, {"dim": 10}, {"scaling": "other"},
                                    {"base": 0.0}, {"base": math.nan}, {"scaling": "linear", "factor": 0.0},
                                    {"scaling": "parts", "factor": 2.0}, {"scaling": "parts", "context": 5.0, "fast": 1.0}])
def test_rotary_refuses(kwargs):
    with pytest.raises(InvalidInput):
        Rotary(8, device=_HostDevice(), **kwargs)


def test_rotary_takes_frequencies():
    dev = _HostDevice()
    assert np.array_equal(Rotary(8, freqs=[1, 2, 3, 4], device=dev).freqs, [1.0, 2.0, 3.0, 4.0])
    with pytest.raises(ShapeMismatch):
        Rotary(8, freqs=[1, 2, 3], device=dev)


def test_tensor_rotary_refuses():
    dev = _HostDevice()
    r = Rotary(8, dim=4, device=dev)
    x = Tensor.empty([2, 3, 5, 8], dev)
    RotaryPositions(x, r)
    RotaryPositions(x, r, positions=np.zeros((2, 5), np.int64))
    RotaryPositions(x, r, positions=np.zeros((2, 3), np.int64), heads_last=True)
    with pytest.raises(InvalidOperation):
        RotaryPositions(Tensor.empty([2, 3, 8], dev), r)
    for bad in (Tensor.empty([2, 3, 5, 4], dev), Tensor.empty([2, 3, 5, 16], dev)):
        with pytest.raises(ShapeMismatch):
            RotaryPositions(bad, r)
    for bad in (np.zeros((2, 3), np.int32), np.zeros(10, np.int32)):
        with pytest.raises(ShapeMismatch):
            RotaryPositions(x, r, positions=bad)
    for bad in (np.zeros((2, 5)), np.full((2, 5), 2**31), np.full((2, 5), -2**31 - 1)):
        with pytest.raises(InvalidInput):
            RotaryPositions(x, r, positions=bad)
    with pytest.raises(InvalidInput):
        RotaryPositions(x, r, first=2**31)
    with pytest.raises(DeviceError):
        RotaryPositions(x, Rotary(8, device=_HostDevice()))


def test_cache_append_rotary_refuses():
    dev = _HostDevice()
    c = KvCache(1, 8, 4, 2, 8, dev)
    step = c.batch([(c.new_sequence(), 3)])
    r = Rotary(8, device=dev)
    q, k = Tensor.empty([3, 4, 8], dev), Tensor.empty([3, 2, 8], dev)
    for bad in ((Tensor.empty([2, 4, 8], dev), k, k), (Tensor.empty([3, 4, 4], dev), k, k), (Tensor.empty([3, 8], dev), k, k),
                (q, Tensor.empty([3, 4, 8], dev), k), (q, k, Tensor.empty([3, 2, 4], dev))):
        with pytest.raises(ShapeMismatch):
            c.append_rotary(step, 0, r, *bad)
    with pytest.raises(ShapeMismatch):
        c.append_rotary(step, 0, Rotary(16, device=dev), q, k, k)
    with pytest.raises(DeviceError):
        c.append_rotary(step, 0, Rotary(8, device=_HostDevice()), q, k, k)
    with pytest.raises(DeviceError):
        c.append_rotary(step, 0, r, Tensor.empty([3, 4, 8], _HostDevice()), k, k)
    with pytest.raises(InvalidInput):
        c.append_rotary(step, 1, r, q, k, k)
    c.truncate(0, 1)
    with pytest.raises(InvalidOperation):
        c.append_rotary(step, 0, r, q, k, k)


def test_c_refusals():
    lib, E, S, U = N.load(), N.BCH_E_INVALID, N.BCH_E_SHAPE, N.BCH_E_UNSUPPORTED
    x, nul = C.c_void_p(64), None
    row, thin = N.AttnLayout(512, 64, 8), N.AttnLayout(512, 64, 7)

    def plan(dim=8, interleaved=0, freq=64):
        return N.Rotary(dim, interleaved, 1.0, freq)

    def dense(b=2, h=3, s=4, d=8, p=plan(), inverse=0, xl=row, ol=row, src=x, dst=x):
        return lib.bch_rotary(nul, b, h, s, d, p, inverse, 0, None, src, xl, dst, ol)
    assert dense() == E and "ctx is NULL" in N.last_error(None)
    for f in ("b", "h", "s", "d"):
        assert dense(**{f: -1}) == S, f
    assert dense(d=0) == S and dense(p=None) == E
    for dim in (0, 3, -2, 10):
        assert dense(p=plan(dim)) == S, dim
    assert dense(p=plan(interleaved=2)) == E and dense(inverse=2) == E and dense(xl=thin) == E and dense(ol=thin) == E

    def append(kv=None, batch=None, parent=None, p=plan(), h=4, ql=row, ol=row, kl=row, vl=row):
        return lib.bch_kv_append_rotary(nul, kv or _pages(), batch or _batch(), parent, p, h, x, ql, x, ol, x, kl, x, vl)
    assert append() == E and "ctx is NULL" in N.last_error(None)
    assert lib.bch_kv_append_rotary(nul, None, _batch(), None, plan(), 4, x, row, x, row, x, row, x, row) == E
    assert lib.bch_kv_append_rotary(nul, _pages(), None, None, plan(), 4, x, row, x, row, x, row, x, row) == E
    assert append(_pages(page_size=0)) == S and append(batch=_batch(total=-1)) == S and append(h=-1) == S
    assert append(p=None) == E and append(p=plan(10)) == S and append(p=plan(interleaved=-1)) == E
    for f in ("ql", "ol", "kl", "vl"):
        assert append(**{f: thin}) == E and "layout" in N.last_error(None), f
    assert append(h=0, ql=thin, ol=thin) == E and "ctx is NULL" in N.last_error(None)
    assert append(batch=_batch(total=200, max_new=129), parent=x) == U and "drafts" in N.last_error(None)
    assert append(h=2**30) == U
