"""Sampling without a GPU: the model the GPU tests compare with, and the refusals, which come before any device call."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from barracuda_amd import Sample, Sampling, Tensor
from barracuda_amd import _native as N
from barracuda_amd.error import DeviceError, InvalidInput, InvalidOperation, ShapeMismatch
from tests.sample_model import choose, keep
from tests.test_kv_cache_host import _HostDevice


def test_model():
    x = np.log(np.array([1, 4, 2, 4, 1], np.float64)).astype(np.float32)
    ids = lambda *a: keep(x, *a)[0].tolist()
    assert ids(1.0, 0, 1.0, 0.0) == [0, 1, 2, 3, 4]
    assert ids(1.0, 1, 1.0, 0.0) == [1] and ids(1.0, 2, 1.0, 0.0) == [1, 3] and ids(1.0, 4, 1.0, 0.0) == [0, 1, 2, 3]
    assert ids(0.0, 0, 1.0, 0.0) == [1] and ids(1.0, 0, 0.0, 0.0) == [1]
    assert ids(1.0, 0, 0.3, 0.0) == [1] and ids(1.0, 0, 0.6, 0.0) == [1, 3] and ids(1.0, 0, 0.8, 0.0) == [1, 2, 3]
    assert ids(1.0, 3, 0.7, 0.0) == [1, 3] and ids(1.0, 0, 1.0, 0.4) == [1, 2, 3] and ids(1.0, 0, 1.0, 1.0) == [1, 3]
    assert choose(x, 0.0, 1.0, 0, 1.0, 0.0)[0] == 0 and choose(x, 0.1, 1.0, 0, 1.0, 0.0)[0] == 1
    assert choose(x, 0.99, 1.0, 0, 1.0, 0.0)[0] == 4 and choose(x, 0.45, 1.0, 2, 1.0, 0.0)[0] == 1
    assert choose(np.full(3, -np.inf, np.float32), 0.5, 1.0, 0, 1.0, 0.0)[:2] == (-1, 0.0)
    assert choose(np.array([-np.inf, np.nan, 0.0], np.float32), 0.0, 1.0, 0, 1.0, 0.0)[0] == 2


@pytest.mark.parametrize("kwargs", [{"temperature": -1.0}, {"temperature": math.nan}, {"top_k": -1}, {"top_k": 1.5}, {"top_k": math.inf}, {"top_p": 1.1},
                                    {"top_p": -0.1}, {"top_p": math.nan}, {"min_p": 1.5}, {"min_p": -1.0}, {"min_p": math.nan}])
def test_rules_refuse(kwargs):
    with pytest.raises(InvalidInput):
        Sampling(**kwargs)


def test_sample_refuses():
    dev = _HostDevice()
    x = Tensor.empty([3, 10], dev)
    Sample(x, [0.0, 0.5, 0.99])
    Sample(x, Tensor.empty([3], dev), [Sampling()] * 3)
    for bad in (Tensor.empty([10], dev), Tensor.empty([1, 3, 10], dev), Tensor.empty([3, 0], dev)):
        with pytest.raises(InvalidOperation):
            Sample(bad, [0.0] * 3)
    for bad in ([0.0], [[0.0] * 3], Tensor.empty([4], dev)):
        with pytest.raises(ShapeMismatch):
            Sample(x, bad)
    for bad in ([0.0, -0.1, 0.0], [0.0, 1.5, 0.0], [0.0, math.nan, 0.0]):
        with pytest.raises(InvalidInput):
            Sample(x, bad)
    for bad in ([Sampling()] * 2, [None] * 3):
        with pytest.raises(InvalidInput):
            Sample(x, [0.0] * 3, bad)
    with pytest.raises(DeviceError):
        Sample(x, Tensor.empty([3], _HostDevice()))
    assert Sample(Tensor.empty([0, 10], dev), []).execute().tokens().size == 0


def test_c_refusals():
    lib, E, S, U = N.load(), N.BCH_E_INVALID, N.BCH_E_SHAPE, N.BCH_E_UNSUPPORTED
    x = C.c_void_p(64)

    def sample(rows=2, vocab=10, stride=10, rule=N.Sampling(1.0, 0, 1.0, 0.0), each=None):
        return lib.bch_sample(None, rows, vocab, x, stride, rule, each, x, x, None)
    assert sample() == E and "ctx is NULL" in N.last_error(None)
    assert sample(rows=-1) == S and sample(vocab=0) == S and sample(stride=9) == S
    assert sample(vocab=2**31 - 1, stride=2**31) == U
    assert sample(rule=None) == E and "rule" in N.last_error(None)
    assert sample(rule=None, each=x) == E and "ctx is NULL" in N.last_error(None)
    for bad in ((-1.0, 0, 1.0, 0.0), (math.nan, 0, 1.0, 0.0), (1.0, -1, 1.0, 0.0), (1.0, 0, 1.5, 0.0), (1.0, 0, math.nan, 0.0),
                (1.0, 0, 1.0, -0.5), (1.0, 0, 1.0, 2.0)):
        assert sample(rule=N.Sampling(*bad)) == E and "must not be negative" in N.last_error(None), bad
