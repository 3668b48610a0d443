"""Rows that sampling's lists or bins decide are decided there: they take about the time of others of their kind, not that of a search
of the whole row by one workgroup."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Sampling, Tensor
from tests.sample_model import keep
from tests.test_gpu_kv_cache import _p, _t
from tests.test_gpu_sample import check

pytestmark = pytest.mark.gpu


def time_of(dev, x, rule):
    """us a call, the least of several runs of calls; the tokens are checked."""
    rows, vocab = x.shape
    rng = np.random.default_rng(vocab)
    u = rng.random(rows, dtype=np.float32)
    tx, tu, to, tp = _t(x, dev), _t(u, dev), Tensor.empty([rows], dev), Tensor.empty([rows], dev)
    native = rule._native()
    call = lambda: dev.check(dev._lib.bch_sample(dev.ctx, rows, vocab, _p(tx), vocab, native, None, _p(tu), _p(to), _p(tp)), "sample")
    events = [C.c_void_p(), C.c_void_p()]
    for e in events:
        dev.check(dev._lib.bch_event_create(dev.ctx, C.byref(e)), "event")
    best = np.inf
    for _ in range(12):
        dev.check(dev._lib.bch_event_record(dev.ctx, events[0]), "event")
        for _ in range(20):
            call()
        dev.check(dev._lib.bch_event_record(dev.ctx, events[1]), "event")
        ms = C.c_float()
        dev.check(dev._lib.bch_event_elapsed_ms(events[0], events[1], C.byref(ms)), "event")
        best = min(best, ms.value * 50)
    for e in events:
        dev._lib.bch_event_destroy(e)
    check(x, u, [rule] * rows, to.to_numpy().view(np.int32), tp.to_numpy())
    return best


def left(rng, rows, vocab, n, lowest=None):
    """Rows of n tokens among nothing; lowest: one of them is that."""
    x = np.full((rows, vocab), -np.inf, np.float32)
    for r in x:
        at = rng.permutation(vocab)[:n]
        r[at] = 2 * rng.standard_normal(n, dtype=np.float32)
        if lowest is not None:
            r[at[0]] = lowest
    return x


@pytest.mark.parametrize("n", [260, 300, 600])
@pytest.mark.parametrize("rule,like", [(Sampling(1.3, 0, 0.98), 100), (Sampling(1.0, 200, 0.9), 1000)])
def test_rows_whose_tokens_are_all_listed(dev, n, rule, like):
    """A few hundred tokens that a mask leaves, fewer in a span than its list would hold."""
    rng = np.random.default_rng(n)
    # (a search of the row, or two further kernels, would make it 2 to 8 times)
    assert time_of(dev, left(rng, 16, 50021, n), rule) <= 1.7 * time_of(dev, left(rng, 16, 50021, like), rule)


@pytest.mark.parametrize("lowest", [-1e4, -1e30, -3.4e38])
def test_an_outlier_does_not_spoil_the_bins_of_weights(dev, lowest):
    rng = np.random.default_rng(5)
    rule = Sampling(1.3, 0, 0.98)
    assert time_of(dev, left(rng, 16, 50021, 500, lowest), rule) <= 1.7 * time_of(dev, left(rng, 16, 50021, 100), rule)


@pytest.mark.parametrize("vocab", [8195, 20001, 50021, 50257, 151936, 200000])
@pytest.mark.parametrize("back", [1, 4])
def test_a_row_whose_last_logits_lie_at_the_cut(dev, vocab, back):
    """Thousands of tokens stay; one that lies where top_p cuts is among the row's last four, or none of those is near."""
    rng = np.random.default_rng(vocab)
    rule = Sampling(1.3, 0, 0.98)
    x = 2 * rng.standard_normal((16, vocab), dtype=np.float32)
    x[:, -4:] = 0.0
    far = time_of(dev, x, rule)
    for r in x:
        ids, _, _ = keep(r, rule.temperature, rule.top_k, rule.top_p, rule.min_p)
        r[-back] = r[ids].min()
    # (a search of the row would add 60 us and more to 40 to 60)
    assert time_of(dev, x, rule) <= 1.4 * far
