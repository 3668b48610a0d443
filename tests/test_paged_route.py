"""Which kernels attention over a paged cache takes (bch_sdpa_paged_kernel_name), without a GPU: no pointer here is
ever followed."""
from __future__ import annotations

import re

from barracuda_amd import _native as N


def kernels(b, total, max_new, max_len, h, hkv, d, window=0, sinks=0):
    """{kernel: (rows, shares, least blocks a share)}, shares 0 where lists are taken whole, -n where n workgroups
    have them dealt out."""
    lay = N.AttnLayout(64 * hkv * d, 64 * d, d)
    kv = N.KvPages(16, 16, lay, lay, 1 << 20, 64, hkv, d, 16, max(1, -(-max_len // 64)))
    text = N.load().bch_sdpa_paged_kernel_name(kv, N.KvBatch(b, total, max_new, max_len, 16, 16), h, window, sinks).decode()
    out = {}
    for part in text.split(" + ") if text else []:
        m = re.fullmatch(r"sdpa_paged_(\w+)_kernel(?: rows=(\d+)(?: whole| dealt=(\d+)| shares=(\d+) least=(\d+)))?", part)
        if m is None:
            assert part == "paged_combine", text
            out["combine"] = True
        else:
            out[m[1]] = (int(m[2] or 0), int(m[4] or 0) - int(m[3] or 0), int(m[5] or 0))
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


def test_short_sequences_have_a_kernel_wherever_long_ones_have_theirs():
    """From 2.8 million sequences on, a workgroup for each list of the few rows' kernel would be more than a grid
    holds, when one for each tile is not: both kernels run, and lists are dealt out."""
    for b in (2796202, 2796203, 3000000, 8388607, 8388608, 1 << 24):
        k = kernels(b, b + 15, 16, 8, 8, 1, 8)
        assert "tile" in k and "rows" in k, (b, k)


def test_a_long_chunk_beside_many_sequences_keeps_its_kernels():
    """Batch times row blocks of the longest chunk beyond a grid, whatever rows there are."""
    for b, new, h, hkv, d, name in ((8192, 8192, 32, 4, 8, "tile"), (1024, 65536, 32, 8, 128, "tile"),
                                    (4096, 1 << 20, 32, 8, 128, "tile"), (1024, 65536, 32, 8, 256, "wide"),
                                    (1 << 20, 1 << 20, 8, 8, 4, "rows")):
        k = kernels(b, new + b - 1, new, new, h, hkv, d)
        assert name in k and "rows" in k and "any" not in k, (b, new, k)


def test_more_sequences_than_a_call_takes_have_no_kernels():
    assert kernels((1 << 24) + 1, 1 << 25, 1, 8, 8, 1, 8) == {}
