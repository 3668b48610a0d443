"""4-bit weights without a GPU: quantization and its inverse on the host, and the refusals, which come before any device call."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Tensor
from barracuda_amd import _native as N
from barracuda_amd.error import DeviceError, InvalidInput, ShapeMismatch
from barracuda_amd.nn import Weights4, dequantize4, linear4, quantize4
from tests.test_kv_cache_host import _HostDevice


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 7, 32), (5, 64, 32), (4, 130, 64), (2, 257, 128), (3, 100, 4096)])
def test_quantize4(n, k, group, zeros):
    rng = np.random.default_rng(1)
    w = rng.standard_normal((n, k)).astype(np.float32) + (2.0 if zeros else 0.0)
    codes, scales, zero = quantize4(w, group, zeros)
    groups = -(-k // group)
    assert codes.shape == (n, -(-k // 2)) and codes.dtype == np.uint8 and scales.shape == (n, groups)
    assert (zero is not None) == zeros
    back = dequantize4(codes, scales, group, k, zero)
    half = np.repeat(scales, group, 1)[:, :k] * (1.0 if zeros else 0.5)  # a zero point is rounded too
    assert np.all(np.abs(back - w) <= half * (1 + 2.0**-20))
    if k % 2:
        assert np.all(codes[:, -1] >> 4 == 0)


def test_quantize4_exact_and_empty_groups():
    w = np.zeros((2, 96), np.float32)
    w[0, 32:64] = np.arange(32) % 15 - 7
    for zeros in (False, True):
        codes, scales, zero = quantize4(w, 32, zeros)
        back = dequantize4(codes, scales, 32, 96, zero)
        assert np.all(back[:, :32] == 0) and np.all(back[1] == 0) and np.all(scales[1] == 0)
        if not zeros:
            assert np.array_equal(back, w)
    for bad in (np.zeros(3), np.zeros((0, 3)), np.full((2, 3), np.nan), np.full((2, 3), np.inf)):
        with pytest.raises(InvalidInput):
            quantize4(bad)
    for group in (0, -32, 16, 33):
        with pytest.raises(InvalidInput):
            quantize4(w, group)


def test_weights_refuse():
    dev = _HostDevice()
    ok = dict(codes=np.zeros((4, 33), np.uint8), scales=np.zeros((4, 3), np.float32), in_features=65, group=32)

    def make(**k):
        return Weights4(**{**ok, "device": dev, **k})
    for bad in (dict(codes=np.zeros((4, 32), np.uint8)), dict(codes=np.zeros((4, 33), np.int8)), dict(codes=np.zeros(33, np.uint8)),
                dict(codes=np.zeros((0, 33), np.uint8)), dict(in_features=0), dict(group=0), dict(group=48),
                dict(zeros=np.full((4, 3), 16)), dict(zeros=np.full((4, 3), -1)), dict(zeros=np.zeros((4, 3)))):
        with pytest.raises(InvalidInput):
            make(**bad)
    for bad in (dict(scales=np.zeros((4, 2), np.float32)), dict(zeros=np.zeros((3, 4), np.uint8))):
        with pytest.raises(ShapeMismatch):
            make(**bad)


class _Given:
    """What linear4 asks of Weights4."""

    def __init__(self, dev, n, k):
        from barracuda_amd.tensor import _Buffer
        self.device, self.out_features, self.in_features, self._buf = dev, n, k, _Buffer(dev, 16)


def test_linear4_refuses():
    dev = _HostDevice()
    w = _Given(dev, 5, 40)
    for shape in ([40], [2, 39], [2, 40, 1]):
        with pytest.raises(InvalidInput):
            linear4(Tensor.empty(shape, dev), w)
    with pytest.raises(InvalidInput):
        linear4(Tensor.empty([2, 40], dev), w, Tensor.empty([4], dev))
    with pytest.raises(DeviceError):
        linear4(Tensor.empty([2, 40], _HostDevice()), w)
    assert linear4(Tensor.empty([0, 40], dev), w).shape() == [0, 5]


def test_c_refusals():
    lib, E, S, U = N.load(), N.BCH_E_INVALID, N.BCH_E_SHAPE, N.BCH_E_UNSUPPORTED
    size, x, odd = C.c_size_t(), C.c_void_p(64), C.c_void_p(72)
    assert lib.bch_w4_bytes(17, 129, 128, C.byref(size)) == 0 and size.value == 2 * 2 * 1024 + 80 * 2 * 2
    assert lib.bch_w4_bytes(16, 128, 2**31 - 32, C.byref(size)) == 0 and size.value == 1024 + 80
    assert lib.bch_w4_bytes(2**26 - 16, 4096, 128, C.byref(size)) == 0 and size.value == (2**22 - 1) * 32 * (1024 + 80)
    assert lib.bch_w4_bytes(17, 129, 128, None) == E
    for n, k, g, st in ((0, 1, 32, S), (1, 0, 32, S), (1, 1, 0, S), (-1, 1, 32, S), (1, 1, 33, E), (1, 1, 16, E),
                        (2**26 - 15, 1, 32, U), (1, 2**31 - 1, 32, U)):
        assert lib.bch_w4_bytes(n, k, g, C.byref(size)) == st, (n, k, g)
        assert lib.bch_w4_pack(None, n, k, g, x, 2**31 - 1, x, None, x) == st, (n, k, g)
        assert lib.bch_w4_linear(None, 1, N.W4(n, k, g, 64), x, 2**31 - 1, None, 0, x, 2**31 - 1) == st, (n, k, g)
    assert lib.bch_w4_pack(None, 4, 9, 32, x, 4, x, None, x) == S
    assert lib.bch_w4_pack(None, 4, 9, 32, x, 5, x, None, x) == E and "ctx is NULL" in N.last_error(None)
    w = N.W4(4, 9, 32, 64)

    def linear(m=3, w=w, ldx=9, act=0, ldy=4):
        return lib.bch_w4_linear(None, m, w, x, ldx, None, act, x, ldy)
    assert linear() == E and "ctx is NULL" in N.last_error(None)
    assert linear(w=None) == E and linear(act=3) == E and linear(act=-1) == E
    assert linear(m=-1) == S and linear(ldx=8) == S and linear(ldy=3) == S
