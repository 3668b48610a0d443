"""Attention over a paged cache for 17 to 48 rows a sequence and key/value head over long lists of keys, where a
workgroup takes 32 rows, against plain forms in 64 bits.  Short sequences beside them make the lists long enough
together."""
import numpy as np
import pytest

from tests.test_gpu_paged import Case, _tree

pytestmark = pytest.mark.gpu


def _beside(d, lens, news):
    n = 80 if d <= 64 else 30
    return lens + [1 + i % 5 for i in range(n)], news + [1] * n


@pytest.mark.parametrize("d", [4, 7, 33, 64, 80, 100, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 0), (2500, 40)])
def test_chunks(dev, d, window, sinks):
    for lens, news, h, hkv in (([3300, 2900, 40, 9], [5, 8, 1, 0], 8, 2), ([3000, 2700], [17, 31], 3, 3),
                               ([3100], [48], 1, 1), ([3222, 2800], [2, 1], 48, 2), ([2700, 3600, 20], [32, 33, 16], 2, 2)):
        print(f"pairs d={d} lens={lens} news={news} window={window}", flush=True)
        Case(dev, *_beside(d, lens, news), h, hkv, d, 16, window, sinks).check()


def test_many_sequences(dev):
    lens = [1 + 37 * (i % 70) for i in range(150)]
    news = [min(n, 1 + i % 6) for i, n in enumerate(lens)]
    Case(dev, lens, news, 16, 2, 64, 16).check()
    Case(dev, lens, news, 8, 1, 128, 16, 1500, 4).check()


@pytest.mark.parametrize("window,sinks", [(0, 0), (3, 2900), (2200, 4)])
@pytest.mark.parametrize("d", [50, 64, 100, 128])
def test_tree(dev, d, window, sinks):
    rng = np.random.default_rng(d + window)
    for lens, news, h, hkv in (([3000, 2777, 900], [8, 12, 5], 8, 2), ([2800, 60], [40, 33], 2, 2)):
        lens, news = _beside(d, lens, news)
        for deep in (False, True):
            print(f"pairs tree d={d} lens={lens[:3]} window={window} deep={deep}", flush=True)
            Case(dev, lens, news, h, hkv, d, 16, window, sinks, parents=[_tree(rng, n, deep) for n in news]).check()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("d", [64, 100, 128])
def test_values_behind_the_mask_do_not_reach_a_row(dev, d, bad):
    """Keys that some rows of a block see and others do not hold `bad`, and so does all that is not a key."""
    long, page = [2900, 2645, 30], 16
    lens, news = _beside(d, long, [12, 9, 12])
    c = Case(dev, lens, news, 8, 2, d, page, 2100, 2, fill=bad)
    c.check()
    for b, length in enumerate(long):
        for j in (length - 1, length - 5, length - 2104):
            if j > 0:
                c.pool.v[c.pool.table[b, j // page], 0, j % page, ::3] = bad
                c.pool.k[c.pool.table[b, j // page], 1, j % page, [1, d - 2]] = bad
    c.upload()
    c.check()


@pytest.mark.parametrize("d", [64, 128])
def test_pages_not_held_and_rows_before_the_first_key(dev, d):
    c = Case(dev, *_beside(d, [2400, 2300, 3], [10, 12, 9]), 8, 2, d, 16)
    c.pool.table[0, [0, 3, 7, 86]] = [-1, c.pool.num, 2**31 - 1, -2**31]
    c.pool.table[1, :] = -1
    c.upload()
    got = c.check()
    assert np.all(got[10:22] == 0) and np.all(got[22:28] == 0)
