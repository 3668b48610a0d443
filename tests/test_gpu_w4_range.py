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
