"""Rotary positions in 64 bits on the host, for the tests."""
from __future__ import annotations

import numpy as np

# Of scale * (|a| + |b|), what a turned value may be off by: cosine and sine by 1.6 * 2^-24 each (the angle's remainder
# rounded, 2^-25; Taylor's series cut, 2^-28; its last two operations, 2^-25 each) and 2^-24 for `scale`; the product and the sum
# 2^-24 each.  Rounded up.
BOUND = 5 * 2.0**-24


def turned(x, positions, freqs, dim, interleaved, scale, inverse=False):
    """(values, bound): x [..., D] turned, positions broadcast against x's leading axes."""
    x = np.asarray(x, dtype=np.float64)
    t = np.asarray(positions, dtype=np.float64)[..., None] * freqs * (-1 if inverse else 1)
    c, s = scale * np.cos(t), scale * np.sin(t)
    i = np.arange(dim // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)
    y, bound = x.copy(), np.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    bound[..., a] = bound[..., b] = BOUND * abs(scale) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, bound


def depths(parents):
    out = []
    for i, p in enumerate(parents):
        out.append(out[p] + 1 if 0 <= p < i else 0)
    return out
