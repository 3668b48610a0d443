"""Which kernels attention over a paged cache takes (bch_sdpa_paged_kernel_name), without a GPU: no pointer here is
ever followed."""
from __future__ import annotations

import re

from barracuda_amd import _native as N


def kernels(b, total, max_new, max_len, h, hkv, d, window=0, sinks=0):
    """{kernel: (rows, shares, least blocks a share)}, shares 0 where lists are taken whole."""
    lay = N.AttnLayout(64 * hkv * d, 64 * d, d)
    kv = N.KvPages(16, 16, lay, lay, 1 << 20, 64, hkv, d, 16, max(1, -(-max_len // 64)))
    text = N.load().bch_sdpa_paged_kernel_name(kv, N.KvBatch(b, total, max_new, max_len, 16, 16), h, window, sinks).decode()
    out = {}
    for part in text.split(" + ") if text else []:
        m = re.fullmatch(r"sdpa_paged_(\w+)_kernel(?: rows=(\d+)(?: (whole)| shares=(\d+) least=(\d+)))?", part)
        if m is None:
            assert part == "paged_combine", text
            out["combine"] = True
        else:
            out[m[1]] = tuple(int(x or 0) for x in (m[2], m[4], m[5]))
    return out


def test_kernels_by_width_and_rows():
    assert kernels(2, 2, 1, 300, 8, 8, 64) == {"rows": (16, 0, 0)}
    assert kernels(1, 5, 5, 40, 4, 2, 3) == {"any": (0, 0, 0)}
    assert kernels(1, 5, 5, 40, 4, 2, 300) == {"any": (0, 0, 0)}
    assert {"tile", "rows"} <= set(kernels(4, 4000, 1000, 1000, 8, 2, 128))
    assert "wide" in kernels(4, 4000, 1000, 1000, 8, 2, 192)
    k = kernels(4, 4, 1, 65536, 32, 8, 128)
    assert k["combine"] and k["rows"][1] > 0


def test_calls_that_launch_nothing_have_no_kernels():
    assert kernels(0, 0, 0, 0, 8, 8, 64) == {} and kernels(2, 0, 0, 40, 8, 8, 64) == {}
    assert kernels(2, 2, 1, 40, 7, 2, 64) == {} and kernels(2, 2, 1, 40, 2, 2, 2000) == {}
    assert N.load().bch_sdpa_paged_kernel_name(None, None, 1, 0, 0) == b""
