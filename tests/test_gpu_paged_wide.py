"""Attention over a paged cache for many rows of 129 to 256 floats, against plain forms in 64 bits."""
import numpy as np
import pytest

from tests.test_gpu_paged import Case, _tree, compare, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [129, 131, 160, 191, 192, 193, 250, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 3), (70, 4000), (200, 33)])
def test_chunks(dev, d, window, sinks):
    for lens, news, h, hkv, page in (([70, 33, 400, 9], [70, 1, 131, 0], 4, 2, 16), ([150, 290], [129, 290], 3, 1, 7)):
        print(f"wide d={d} lens={lens} news={news} window={window} sinks={sinks}", flush=True)
        Case(dev, lens, news, h, hkv, d, page, window, sinks).check()


@pytest.mark.parametrize("n", [12, 13, 31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129])
@pytest.mark.parametrize("d", [192, 256])
def test_every_block_edge(dev, n, d):
    """Rows and keys on either side of the blocks: 4 and 1 rows a token."""
    for h, hkv in ((4, 1), (2, 2)):
        for more in (0, 1, 40):
            print(f"wide edge n={n} d={d} h={h} more={more}", flush=True)
            Case(dev, [n + more, 2 * n], [n, n], h, hkv, d, 16, 24, 2).check()


@pytest.mark.parametrize("d", [150, 256])
def test_long_lists_and_many_tiles(dev, d):
    """Lists cut over workgroups, lists taken whole."""
    Case(dev, [3000, 700, 5], [20, 600, 5], 4, 1, d, 64).check()
    Case(dev, [3000, 700], [20, 600], 4, 1, d, 64, 333, 70).check()
    Case(dev, [520] * 4, [510] * 4, 16, 2, d, 32, 100, 1).check()


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("row_pad,misalign", [(0, 0), (3, 0), (0, 1), (4, 2)])
def test_strides_and_alignment(dev, row_pad, misalign, slots):
    for d in (192, 253):
        Case(dev, [333, 140], [100, 140], 6, 2, d, 16, 100, 2, row_pad=row_pad, misalign=misalign, slots=slots).check()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("d", [131, 192, 256])
def test_values_behind_the_mask_do_not_reach_a_row(dev, d, bad):
    """Everything in the pool that is not a key is `bad`, and so are keys that some rows see and others do not."""
    lens, news, page = [170, 45, 300], [50, 45, 130], 16
    c = Case(dev, lens, news, 4, 2, d, page, 20, 2, fill=bad)
    c.check()
    for b, (length, n) in enumerate(zip(lens, news)):
        for j in (length - 1, length - 30, length - 41):
            c.pool.v[c.pool.table[b, j // page], 0, j % page, ::3] = bad
            c.pool.k[c.pool.table[b, j // page], 1, j % page, [1, d - 2]] = bad
    c.upload()
    c.check()


def test_pages_not_held(dev):
    c = Case(dev, [400, 300], [30, 200], 4, 2, 256, 16)
    c.pool.table[0, [0, 3, 7, 24]] = [-1, c.pool.num, 2**31 - 1, -2**31]
    c.upload()
    c.check()
    c.pool.table[1, :] = -1
    c.upload()
    assert np.all(c.check()[30:] == 0)


def test_extreme_queries(dev):
    c = Case(dev, [200, 90], [60, 33], 4, 2, 200, 16, 40, 2)
    c.q[0, 1, 3] = np.nan
    c.q[c.total - 1, 2, 0] = np.inf
    c.upload()
    dev.check(c.call(dev._lib, dev.ctx), "attention")
    got, want = c.output(), c.want()
    rows = np.ones(c.total, bool)
    rows[[0, c.total - 1]] = False
    compare(got[rows], want[rows], tolerance(c.q[:c.total][rows], c.pool.k, c.pool.v, c.scale, 200))
    assert np.all(np.isnan(got[0, 1])) and np.all(np.isnan(got[c.total - 1, 2]))
    assert np.all(np.isfinite(got[0, [0, 2, 3]]))


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 0), (2, 300), (40, 4)])
@pytest.mark.parametrize("d", [140, 256])
def test_tree(dev, d, window, sinks):
    rng = np.random.default_rng(d + window)
    for lens, news in (([500, 77], [16, 60]), ([300, 64, 200], [64, 64, 0]), ([200, 1700], [128, 100]), ([140], [128])):
        for deep in (False, True):
            print(f"wide tree lens={lens} news={news} d={d} window={window} deep={deep}", flush=True)
            Case(dev, lens, news, 4, 1, d, 16, window, sinks, parents=[_tree(rng, n, deep) for n in news]).check()


def test_more_rows_than_keys(dev):
    got = Case(dev, [3, 0, 5], [40, 30, 5], 4, 2, 256, 16, 2, 1).check()
    assert np.all(got[:37] == 0) and np.all(got[40:70] == 0)
    lens, news = [5, 290], [200, 290]
    a = Case(dev, lens, news, 4, 2, 192, 16).check()
    for window in (290, 2**31 - 1):
        assert np.array_equal(Case(dev, lens, news, 4, 2, 192, 16, window).check(), a)
