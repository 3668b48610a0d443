"""Linear layers of 4-bit weights on the GPU against 64 bits: sizes and groups around the kernels' tiles, strides,
special values, and what has to be exact."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Tensor
from barracuda_amd import _native as N
from barracuda_amd.nn import Activation, Weights4, dequantize4, linear4, quantize4
from oracle import bc_oracle as O
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip
from tests.test_gpu_kv_cache import _p, _t

pytestmark = pytest.mark.gpu


def weights(rng, n, k, group, zeros):
    groups = -(-k // group)
    codes = rng.integers(0, 256, (n, -(-k // 2)), dtype=np.uint8)
    scales = (rng.random((n, groups), dtype=np.float32) + 0.5) * np.float32(0.1)
    return codes, scales, rng.integers(0, 16, (n, groups), dtype=np.uint8) if zeros else None


def wide(codes, scales, group, k, zeros):
    """The weights in 64 bits."""
    code = np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)[:, :k].astype(np.float64)
    pick = np.arange(k) // group
    return scales.astype(np.float64)[:, pick] * (code - (8.0 if zeros is None else zeros.astype(np.float64)[:, pick]))


def slack(x, w, bias=None):
    """Products are exact or rounded once, a group's sum once more by its scale; the sums of k products have at most 3 k / 16 +
    32 additions one behind the other (three parts of 16 inputs an instruction, or 8 and then one a group of a lane), each off by
    2^-24 of what has been added up in magnitude; the bias is one more."""
    x, w = np.abs(x.astype(np.float64)), np.abs(w)
    total = x @ w.T
    if bias is not None:
        total = total + np.abs(bias)
    return (3 * x.shape[1] / 16 + 34) * 2.0**-24 * total


def check(dev, rng, m, n, k, group, zeros, bias=False, act=None, x=None):
    c, s, z = weights(rng, n, k, group, zeros)
    x = rng.standard_normal((m, k), dtype=np.float32) if x is None else x
    b = rng.standard_normal(n, dtype=np.float32) if bias else None
    got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev), _t(b, dev) if bias else None, act).to_numpy()
    w = wide(c, s, group, k, z)
    y = x.astype(np.float64) @ w.T + (b if bias else 0.0)
    tol = slack(x, w, b)
    if act is Activation.ReLU:
        y = np.maximum(y, 0.0)
    if act is Activation.GELU:
        with np.errstate(over="ignore"):
            y = y / (1.0 + np.exp(-2.0 * 0.7978845608 * (y + 0.044715 * y**3)))
        tol = 1.13 * tol + 8 * 2.0**-24 * np.abs(y) + 1e-37  # GELU's slope is at most 1.13; its own roundings
    worst = np.max(np.abs(got - y) - tol)
    assert worst <= 0, (worst, np.unravel_index(np.argmax(np.abs(got - y) - tol), y.shape))


MS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129, 200, 257]


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k,group,zeros", [(1, 1, 32, False), (16, 128, 128, True), (17, 129, 32, True), (50, 100, 64, False),
                                             (130, 300, 96, True), (257, 513, 256, True), (64, 1000, 1024, False),
                                             (300, 31, 32, True), (33, 1025, 160, False)])
def test_sizes(dev, m, n, k, group, zeros):
    check(dev, np.random.default_rng(m), m, n, k, group, zeros, bias=m % 2 == 0)


@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 11008, 4096, 128, False), (3, 4096, 11008, 128, True), (16, 2999, 4099, 64, True),
                                               (32, 4096, 4096, 32, False), (64, 1031, 8192, 128, True), (96, 2048, 2048, 128, False),
                                               (300, 1000, 4096, 64, True), (513, 769, 1500, 128, False), (1, 5, 20000, 128, True),
                                               (8, 40, 30001, 32, True), (700, 20, 9000, 128, False), (2048, 512, 512, 128, True)])
def test_large(dev, m, n, k, group, zeros):
    check(dev, np.random.default_rng(3), m, n, k, group, zeros)


@pytest.mark.parametrize("m", [1, 5, 12, 40, 70, 300])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("act", [Activation.ReLU, Activation.GELU])
def test_epilogue(dev, m, bias, act):
    check(dev, np.random.default_rng(4), m, 77, 200, 64, True, bias, act)


@pytest.mark.parametrize("m", MS)
def test_whole_numbers_are_exact(dev, m):
    rng = np.random.default_rng(5)
    n, k, group = 100, 700, 64
    c, _, z = weights(rng, n, k, group, True)
    s = np.float32(2.0) ** rng.integers(-2, 3, (n, -(-k // group))).astype(np.float32)
    x = rng.integers(-100, 101, (m, k)).astype(np.float32)
    got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
    assert np.array_equal(got, x.astype(np.float64) @ wide(c, s, group, k, z).T)


@pytest.mark.parametrize("m", MS)
def test_one_product_alone(dev, m):
    """Rows with one input that is not zero, over the magnitudes of f32: x (c - z) s, rounded at most three times."""
    rng = np.random.default_rng(6)
    n, k, group = 48, 333, 32
    c, s, z = weights(rng, n, k, group, True)
    at = rng.integers(0, k, m)
    x = np.zeros((m, k), np.float32)
    x[np.arange(m), at] = np.ldexp(rng.uniform(1, 2, m) * rng.choice([-1, 1], m), rng.integers(-120, 120, m))
    got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
    want = x.astype(np.float64) @ wide(c, s, group, k, z).T
    assert np.all(np.abs(got - want) <= 3 * 2.0**-24 * np.abs(want) + 2.0**-149)


@pytest.mark.parametrize("m", [1, 6, 16, 33, 80, 300])
def test_small_beside_large(dev, m):
    """An input 2^60 times the others whose weights are at their zero point does not reach the sum."""
    rng = np.random.default_rng(7)
    n, k, group = 32, 256, 64
    c, s, z = weights(rng, n, k, group, False)
    code = np.stack([c & 15, c >> 4], 2).reshape(n, -1)
    code[:, 77] = 8
    c = code[:, 0::2] | (code[:, 1::2] << 4)
    x = rng.standard_normal((m, k), dtype=np.float32)
    y = x.copy()
    y[:, 77] = 2.0**60
    w = Weights4(c, s, k, group, None, dev)
    a, b = linear4(_t(x, dev), w).to_numpy(), linear4(_t(y, dev), w).to_numpy()
    x[:, 77] = 0
    tol = slack(x, wide(c, s, group, k, None))
    assert np.all(np.abs(b - a) <= 2 * tol)


@pytest.mark.parametrize("m", [1, 3, 16, 33, 80, 300])
def test_zero_weights_and_zero_rows(dev, m):
    rng = np.random.default_rng(8)
    n, k, group = 40, 200, 32
    z = rng.integers(0, 16, (n, -(-k // group)), dtype=np.uint8)
    code = np.repeat(z, group, 1)[:, :k]
    c = (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)
    s = np.ones((n, z.shape[1]), np.float32)
    x = rng.standard_normal((m, k), dtype=np.float32) * np.float32(1e30)
    assert np.all(linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy() == 0)
    c, s, z = weights(rng, n, k, group, True)
    b = rng.standard_normal(n, dtype=np.float32)
    got = linear4(_t(np.zeros((m, k), np.float32), dev), Weights4(c, s, k, group, z, dev), _t(b, dev)).to_numpy()
    assert np.array_equal(got, np.repeat(b[None], m, 0))


@pytest.mark.parametrize("m", [1, 4, 9, 33, 80, 300])
def test_special_values(dev, m):
    """Infinities and NaN reach the rows that hold them and no other: an infinity times a weight is an infinity of its
    sign, or NaN where the weight is zero."""
    rng = np.random.default_rng(9)
    n, k, group = 64, 160, 32
    c, s, z = weights(rng, n, k, group, True)
    w = wide(c, s, group, k, z)
    x = rng.standard_normal((m, k), dtype=np.float32)
    x[0, 100] = np.inf
    if m > 2:
        x[m - 1, 3], x[m // 2, 159] = np.nan, -np.inf
    b = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
    with np.errstate(invalid="ignore"):
        for i in range(m):
            if np.isnan(x[i]).any():
                assert np.isnan(b[i]).all()
            elif np.isinf(x[i]).any():
                assert np.array_equal(b[i], np.sum(x[i][np.isinf(x[i])][None] * w[:, np.isinf(x[i])], 1).astype(np.float32),
                                      equal_nan=True)
            else:
                assert np.all(np.abs(b[i] - x[i].astype(np.float64) @ w.T) <= slack(x[i:i + 1], w)[0])


@pytest.mark.parametrize("m", [1, 9, 33, 80, 300])
@pytest.mark.parametrize("magnitude", [1e-44, 1e-38, 1e-30, 1e30, 3e35])
def test_magnitudes(dev, m, magnitude):
    """All of f32's magnitudes, beside rows of ordinary ones; results of 2^-149 steps are off by half of one a sum."""
    rng = np.random.default_rng(10)
    n, k, group = 40, 96, 32
    c, s, z = weights(rng, n, k, group, True)
    x = rng.standard_normal((m, k), dtype=np.float32)
    x[0] *= np.float32(magnitude)
    got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
    w = wide(c, s, group, k, z)
    assert np.all(np.abs(got - x.astype(np.float64) @ w.T) <= slack(x, w) + 2.0**-149 * (3 * k))


@pytest.mark.parametrize("m", [1, 2, 9, 33, 80, 300])
@pytest.mark.parametrize("ldx,ldy,shift", [(128, 50, 0), (131, 53, 0), (136, 64, 1), (128, 50, 3)])
def test_strides(dev, m, ldx, ldy, shift):
    rng = np.random.default_rng(11)
    n, k, group = 50, 128, 64
    c, s, z = weights(rng, n, k, group, False)
    whole = rng.standard_normal(shift + m * ldx, dtype=np.float32)
    x = np.lib.stride_tricks.as_strided(whole[shift:], (m, k), (4 * ldx, 4))
    w, tx, ty = Weights4(c, s, k, group, z, dev), _t(whole, dev), _t(np.full(shift + m * ldy, 7.0, np.float32), dev)
    dev.check(dev._lib.bch_w4_linear(dev.ctx, m, w._w, C.c_void_p(tx.ptr + 4 * shift), ldx, None, 0,
                                     C.c_void_p(ty.ptr + 4 * shift), ldy), "linear4")
    y = ty.to_numpy()
    assert np.all(y[:shift] == 7.0)
    y = y[shift:].reshape(m, ldy)
    assert np.all(y[:, n:] == 7.0)
    full = wide(c, s, group, k, z)
    assert np.all(np.abs(y[:, :n] - x.astype(np.float64) @ full.T) <= slack(x, full))


def test_quantized_layer(dev):
    """Weights4.quantize of a Tensor against linear over the weights that the codes stand for."""
    rng = np.random.default_rng(12)
    w = rng.standard_normal((70, 300), dtype=np.float32)
    x = rng.standard_normal((5, 300), dtype=np.float32)
    for zeros in (False, True):
        q = Weights4.quantize(_t(w, dev), 64, zeros)
        back = dequantize4(*quantize4(w, 64, zeros)[:2], 64, 300, quantize4(w, 64, zeros)[2])
        got = linear4(_t(x, dev), q).to_numpy()
        assert np.all(np.abs(got - x.astype(np.float64) @ back.astype(np.float64).T) <= slack(x, back) * (1 + 2.0**-20))


@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k,group", [(9001, 200, 64), (8201, 300, 32), (8209, 9000, 160), (16400, 130, 128), (20001, 1, 32)])
def test_one_row_many_outputs(dev, m, n, k, group):
    """More workgroups than the card holds at a time."""
    check(dev, np.random.default_rng(n), m, n, k, group, True, bias=True, act=Activation.ReLU)


@pytest.mark.parametrize("m,n,k,group,zeros,act", [(2050, 20, 5000, 64, True, None), (2056, 36, 4609, 32, False, Activation.ReLU),
                                                   (70, 24, 20001, 32, True, None), (65, 259, 16392, 128, False, Activation.GELU),
                                                   (129, 16, 9000, 96, True, None), (300, 1000, 1000, 32, True, Activation.GELU),
                                                   (65, 64, 40000, 256, False, None), (191, 1030, 2000, 64, False, Activation.ReLU)])
def test_many_rows(dev, m, n, k, group, zeros, act):
    """Rows in fours and in eights with more inputs than a workgroup holds, many slices, and columns that do not fill a tile."""
    check(dev, np.random.default_rng(m + k), m, n, k, group, zeros, bias=True, act=act)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (32, 1024, 8192), (64, 300, 3000), (130, 700, 1024)])
def test_repeats_bit_for_bit_and_under_capture(dev, m, n, k):
    """The same call gives the same bits; captured on a fresh context (no workspace) it gives them to rounding, at every replay."""
    rng = np.random.default_rng(13)
    c, s, z = weights(rng, n, k, 128, True)
    w = Weights4(c, s, k, 128, z, dev)
    x = rng.standard_normal((m, k), dtype=np.float32)
    tx = _t(x, dev)
    first = linear4(tx, w).to_numpy()
    for _ in range(3):
        linear4(_t(x[::-1].copy(), dev), w)
        assert np.array_equal(linear4(tx, w).to_numpy(), first)
    full = wide(c, s, 128, k, z)
    hip = _hip()
    dev.sync()
    with _FreshCtx(dev) as f:
        ty = Tensor.empty([m, n], dev)
        dev.sync()
        call = lambda: f.lib.bch_w4_linear(f.ctx, m, w._w, _p(tx), k, None, 0, _p(ty), n)
        assert hip.hipStreamBeginCapture(f.stream, CAPTURE_RELAXED) == 0
        st = call()
        graph, ex = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamEndCapture(f.stream, C.byref(graph)) == 0 and st == 0
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
        tol = slack(x, full)
        seen = None
        for _ in range(3):
            assert hip.hipGraphLaunch(ex, f.stream) == 0 and f.lib.bch_sync(f.ctx) == 0
            got = ty.to_numpy()
            assert np.all(np.abs(got - x.astype(np.float64) @ full.T) <= tol)
            assert seen is None or np.array_equal(seen, got)
            seen = got
            assert call() == 0 and f.lib.bch_sync(f.ctx) == 0  # an eager call between: its workspace may be new
        assert np.array_equal(ty.to_numpy(), first)
        hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(graph)
