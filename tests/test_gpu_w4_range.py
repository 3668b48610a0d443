"""Linear layers of 4-bit weights at the ends of f32's range, on the GPU against 64 bits: what is finite in f32 stays finite, and
inputs far below others of their row keep their bits, however many rows a call has."""
from __future__ import annotations

import numpy as np
import pytest

from barracuda_amd.nn import Weights4, linear4
from tests.test_gpu_kv_cache import _t
from tests.test_gpu_w4 import slack, weights, wide

pytestmark = pytest.mark.gpu

MS = [1, 2, 3, 9, 33, 64, 65, 80, 300]


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("k,group", [(96, 32), (9000, 128)])
@pytest.mark.parametrize("top", [2.0**20, 2.0**30, 2.0**100, 2.0**116, 2.0**124, 2.0**127 * 1.5])
def test_large_inputs_whose_weights_are_small(dev, m, k, group, top):
    """One or a few inputs up to f32's largest, in the first of the inputs, the last of them, or both: 15 of them would not fit, times
    their scales they do."""
    rng = np.random.default_rng(1)
    n = 40
    c, s, z = weights(rng, n, k, group, True)
    s *= np.float32(0.01)
    w = wide(c, s, group, k, z)
    for at in ([3], [k - 2], [5, k - 1]):
        x = rng.standard_normal((m, k), dtype=np.float32)
        for i in sorted({0, m // 2, m - 1}):
            x[i, at] = np.float32(top) * rng.choice([-1, 1], len(at)).astype(np.float32) / np.float32(len(at))
        want = x.astype(np.float64) @ w.T
        assert np.abs(want).max() < 3e38
        got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
        assert np.all(np.abs(got - want) <= slack(x, w))


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("large", [2.0**60, 2.0**100, 2.0**127 * 1.5, -(2.0**127) * 1.9])
def test_ordinary_inputs_beside_one_whose_weights_are_zero(dev, m, group, large):
    """An input whose weights are all at their zero point leaves the others' sums as they are, however large it is."""
    rng = np.random.default_rng(2)
    n, k = 40, 390
    c, s, z = weights(rng, n, k, group, True)
    code = np.stack([c & 15, c >> 4], 2).reshape(n, -1)
    code[:, 77] = z[:, 77 // group]
    c = code[:, 0::2] | (code[:, 1::2] << 4)
    w = wide(c, s, group, k, z)
    assert np.all(w[:, 77] == 0)
    for small in (1.0, 2.0**-20):
        x = (rng.standard_normal((m, k), dtype=np.float32) * np.float32(small))
        want, tol = x.astype(np.float64) @ w.T, slack(x, w)
        x[0, 77] = x[m - 1, 77] = np.float32(large)
        assert np.all(np.abs(linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy() - want) <= tol)


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("k,group", [(96, 32), (700, 128)])
@pytest.mark.parametrize("x_log,scale_log", [(5, 113), (-20, 125), (-60, 120), (-100, 127), (-140, 100), (-140, 127), (20, -130),
                                             (100, -140), (120, -149), (-30, -100), (-70, -70)])
def test_scales_of_any_magnitude(dev, m, k, group, x_log, scale_log):
    """What inputs and scales of opposite magnitudes give is what f32 gives; results of 2^-149 steps are off by half of one a sum."""
    rng = np.random.default_rng(3)
    n = 40
    c, s, z = weights(rng, n, k, group, True)
    s = np.ldexp(np.float32(1.0), rng.integers(scale_log, scale_log + 1, s.shape)).astype(np.float32)
    x = np.ldexp(rng.integers(-7, 8, (m, k)).astype(np.float32), x_log - 3).astype(np.float32)
    w = wide(c, s, group, k, z)
    want = x.astype(np.float64) @ w.T
    assert np.abs(want).max() < 2.0**127
    got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
    assert np.all(np.abs(got - want) <= slack(x, w) + 2.0**-149 * (3 * k))


@pytest.mark.parametrize("k", [96, 9000])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_two_rows_of_which_one_is_not_finite(dev, k, bad):
    """What is lost before the scale is computed again in a row of finite inputs, whatever the other row holds."""
    rng = np.random.default_rng(4)
    n, group = 40, 32
    c, s, z = weights(rng, n, k, group, True)
    s *= np.float32(0.01)
    w = wide(c, s, group, k, z)
    for at in (0, 1):
        x = rng.standard_normal((2, k), dtype=np.float32)
        x[at, k // 2], x[1 - at, 5] = bad, 3e38
        got = linear4(_t(x, dev), Weights4(c, s, k, group, z, dev)).to_numpy()
        y = x[1 - at].astype(np.float64) @ w.T
        assert np.all(np.abs(got[1 - at] - y) <= slack(x[1 - at:2 - at], w)[0])
        with np.errstate(invalid="ignore"):
            assert np.array_equal(got[at], (np.float32(bad) * w[:, k // 2]).astype(np.float32), equal_nan=True)
