"""Sampling on the GPU against the choice in 64 bits: sizes, rules, equal logits, masks, and numbers on the borders."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import Sampling, Tensor
from barracuda_amd import _native as N
from tests.sample_model import choose, keep, slack
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip
from tests.test_gpu_kv_cache import _p, _t

pytestmark = pytest.mark.gpu

RULES = [Sampling(), Sampling(0.0), Sampling(0.7, 1), Sampling(0.8, 40), Sampling(1.0, 40, 0.9), Sampling(1.0, 0, 0.95),
         Sampling(1.5, 0, 0.5, 0.01), Sampling(1.0, 0, 1.0, 0.1), Sampling(0.3, 5, 0.99, 0.2), Sampling(1.0, 10**9, 0.999),
         Sampling(1e-4), Sampling(100.0, 0, 0.7), Sampling(1.0, 0, 0.0), Sampling(1.0, 0, 1.0, 1.0), Sampling(float("inf"), 0, 0.6),
         Sampling(1.0, 700, 0.97)]


def logits(rng, rows, vocab, kind):
    x = rng.standard_normal((rows, vocab), dtype=np.float32)
    if kind == "peaked":
        x = 2 * x + np.float32(8) * (rng.random((rows, vocab), dtype=np.float32) < 0.01) * rng.random((rows, vocab), dtype=np.float32)
    if kind == "flat":
        x *= np.float32(0.01)
    if kind == "coarse":  # many equal ones
        x = np.round(x * 2) / np.float32(2) * rng.choice(np.array([1, -1], np.float32), (rows, vocab))
    if kind == "equal":
        x[:] = np.float32(-3.25)
    if kind == "masked":
        x[rng.random((rows, vocab)) < 0.95] = -np.inf
        x[rng.random((rows, vocab)) < 0.01] = np.nan
    if kind == "wide":
        x *= np.float32(1e4)
    return x


def check(x, u, rules, got, probs, near=True):
    skipped = 0
    for i in range(len(x)):
        r = rules[i]
        token, p, border = choose(x[i], u[i], r.temperature, r.top_k, r.top_p, r.min_p)
        if border <= slack(x[i], r.temperature):
            skipped += 1  # a border within the weights' rounding: either side may be taken
            ids, w, _ = keep(x[i], r.temperature, r.top_k, r.top_p, r.min_p)
            assert got[i] in ids or not near
            continue
        assert got[i] == token, (i, r, got[i], token)
        assert abs(probs[i] - p) <= 2.0**-24 * p + 2 * slack(x[i], r.temperature), (i, r)
    return skipped


@pytest.mark.parametrize("kind", ["normal", "peaked", "flat", "coarse", "equal", "masked", "wide"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 65, 1000, 1024, 1025, 4097, 16384, 20011, 50021, 131072])
def test_rules(dev, vocab, kind):
    rng = np.random.default_rng(vocab)
    rules = RULES if vocab < 100000 else RULES[::3] + [RULES[5]]
    rows = len(rules)
    x = logits(rng, rows, vocab, kind)
    u = rng.random(rows, dtype=np.float32)
    out = _t(x, dev).sample(u, rules)
    skipped = check(x, u, rules, out.tokens(), out.probs.to_numpy())
    assert skipped == 0 or kind in ("equal", "coarse", "flat", "masked")


@pytest.mark.parametrize("rows,vocab", [(1, 200000), (3, 32768), (300, 777), (70, 9000), (257, 64)])
@pytest.mark.parametrize("rule", [Sampling(), Sampling(0.8, 40, 0.95), Sampling(1.2, 0, 0.98)])
def test_batches(dev, rows, vocab, rule):
    rng = np.random.default_rng(rows)
    x, u = logits(rng, rows, vocab, "peaked"), rng.random(rows, dtype=np.float32)
    out = _t(x, dev).sample(u, rule)
    assert check(x, u, [rule] * rows, out.tokens(), out.probs.to_numpy()) == 0


MANY = [Sampling(1.0, k) for k in (2, 20, 50, 200, 255, 256, 257, 700, 2000, 5000)] + [
    Sampling(0.7, 200, 0.9, 0.01), Sampling(1.0, 600, 0.99), Sampling(1.3, 1500, 0.98, 0.05), Sampling(0.7, 0, 0.9), Sampling(1.0, 0, 0.6),
    Sampling(0.5, 0, 0.99, 0.001), Sampling(1.0, 0, 1.0, 0.02), Sampling(2.0, 0, 1.0, 1e-4), Sampling(1.0, 0, 0.9, 1e-6)]


@pytest.mark.parametrize("kind", ["together", "descending", "ascending", "spread", "few"])
@pytest.mark.parametrize("vocab", [9000, 33333, 131072, 300001])
def test_where_the_largest_lie(dev, vocab, kind):
    """The largest logits in one place, in order, or a few hundred among nothing."""
    rng = np.random.default_rng(vocab)
    rows = len(MANY)
    x = rng.standard_normal((rows, vocab), dtype=np.float32)
    if kind == "together":
        x[:, 700:1200] += np.float32(6)
    if kind in ("descending", "ascending"):
        x = np.sort(x, axis=1)[:, ::-1 if kind == "descending" else 1].copy()
    if kind == "spread":
        x *= np.float32(3)
    if kind == "few":
        x[rng.random((rows, vocab)) > 400 / vocab] = -np.inf
    u = rng.random(rows, dtype=np.float32)
    out = _t(x, dev).sample(u, MANY)
    # tokens at a top_p of 0.9 weigh 1e-6 of the whole, those at a min_p of 0.001 lie 5e-8 apart, and slack() is 4e-9 to 2e-8: a row in
    # some hundred lies within it.  Of these it is (by the model alone) one of 131072 tokens in order, top_p 0.9, 2.9e-9 from
    # its border, and one of 300001 spread, min_p 1e-4, 5.3e-9 from its.
    on_border = (vocab == 131072 and kind in ("descending", "ascending")) or (vocab == 300001 and kind == "spread")
    assert check(x, u, MANY, out.tokens(), out.probs.to_numpy()) == on_border


def test_equal_logits_go_by_index(dev):
    """All alike: top_k and top_p take the lowest indexes, and the borders are exact."""
    for vocab in (8, 1000, 30000):
        x = np.full((9, vocab), 2.5, np.float32)
        u = np.arange(9, dtype=np.float32) / 8
        u[8] = np.float32(1 - 2.0**-24)
        for k in (2, 7, vocab // 2):
            got = _t(x, dev).sample(u, Sampling(1.0, k)).tokens()
            assert np.array_equal(got, np.minimum(np.floor(u.astype(np.float64) * k), k - 1)), k
        n = vocab // 2
        got = _t(x, dev).sample(u, Sampling(1.0, 0, 0.5)).tokens()
        assert np.array_equal(got, np.minimum(np.floor(u.astype(np.float64) * n), n - 1))
        assert np.all(_t(x, dev).sample(u, Sampling(0.0)).tokens() == 0)


def test_first_and_last(dev):
    """u of 0 takes the first token with weight, u just below 1 (or, from a buffer, anything from 1 on) the last."""
    x = np.array([[-np.inf, -200.0, 0.0, 1.0, np.nan, -np.inf]] * 6, np.float32)
    u = _t(np.array([0.0, -5.0, np.nan, 1.0, 7.0, np.inf], np.float32), dev)
    assert _t(x, dev).sample(u).tokens().tolist() == [2, 2, 2, 3, 3, 3]  # e^-201 is less than a unit


def test_infinities(dev):
    x = np.array([[0.0, np.inf, 3.0, np.inf], [-np.inf] * 4, [np.nan] * 4, [-np.inf, -np.inf, -3e38, -np.inf],
                  [3e38, -3e38, 3.4e38, np.nan]], np.float32)
    for u, want in ((0.0, [1, -1, -1, 2, 2]), (0.49, [1, -1, -1, 2, 2]), (0.51, [3, -1, -1, 2, 2])):
        out = _t(x, dev).sample([u] * 5)
        assert out.tokens().tolist() == want
        assert out.probs.to_numpy().tolist() == [0.5, 0.0, 0.0, 1.0, 1.0]
    assert _t(x, dev).sample([0.9] * 5, Sampling(0.0)).tokens().tolist() == [1, -1, -1, 2, 2]
    assert _t(x, dev).sample([0.9] * 5, Sampling(2.0, 1)).tokens().tolist() == [1, -1, -1, 2, 2]


def test_negative_zero_is_zero(dev):
    x = np.array([[-0.0, 0.0, -0.0, 0.0]] * 4, np.float32)
    assert _t(x, dev).sample([0.0, 0.3, 0.6, 0.9], Sampling(1.0, 3)).tokens().tolist() == [0, 0, 1, 2]
    assert _t(x, dev).sample([0.9] * 4, Sampling(0.0)).tokens().tolist() == [0] * 4


def test_rules_out_of_range_in_device_memory(dev):
    x = np.log(np.array([[1, 4, 2, 4, 1]] * 7, np.float32))
    rules = np.array([[-1, 0, 1, 0], [np.nan, 0, 1, 0], [1, 0, 7, 0], [1, 0, np.nan, 0], [1, 0, 1, np.nan], [1, 0, 1, 9], [1, 0, -2, 0]],
                     np.float32)
    rules.view(np.int32)[:, 1] = [0, 0, -3, 0, 0, 0, 0]
    tx, tr, tu, to = _t(x, dev), _t(rules, dev), _t(np.full(7, 0.97, np.float32), dev), Tensor.empty([7], dev)
    dev.check(dev._lib.bch_sample(dev.ctx, 7, 5, _p(tx), 5, None, _p(tr), _p(tu), _p(to), None), "sample")
    assert to.to_numpy().view(np.int32).tolist() == [1, 1, 4, 4, 4, 3, 1]


def test_strides_and_alignment(dev):
    rng = np.random.default_rng(5)
    for vocab, stride, shift in ((1000, 1003, 1), (4096, 4100, 0), (4096, 4099, 3), (33, 64, 2)):
        whole = np.full(shift + 6 * stride, 99.0, np.float32)
        x = np.lib.stride_tricks.as_strided(whole[shift:], (6, vocab), (4 * stride, 4))
        x[:] = logits(rng, 6, vocab, "peaked")
        u = rng.random(6, dtype=np.float32)
        t, tu, to, tp = _t(whole, dev), _t(u, dev), Tensor.empty([6], dev), Tensor.empty([6], dev)
        r = N.Sampling(0.9, 30, 0.9, 0.0)
        dev.check(dev._lib.bch_sample(dev.ctx, 6, vocab, C.c_void_p(t.ptr + 4 * shift), stride, r, None, _p(tu), _p(to), _p(tp)),
                  "sample")
        assert check(x, u, [Sampling(0.9, 30, 0.9)] * 6, to.to_numpy().view(np.int32), tp.to_numpy()) == 0


def test_a_row_does_not_depend_on_its_batch(dev):
    rng = np.random.default_rng(6)
    x, u = logits(rng, 80, 33000, "peaked"), rng.random(80, dtype=np.float32)
    rules = [RULES[i % len(RULES)] for i in range(80)]
    whole = _t(x, dev).sample(u, rules)
    for rows in ([5], [70, 3, 22], list(range(40))):
        part = _t(x[rows], dev).sample(u[rows], [rules[i] for i in rows])
        assert np.array_equal(part.tokens(), whole.tokens()[rows])
        assert np.array_equal(part.probs.to_numpy(), whole.probs.to_numpy()[rows])


@pytest.mark.parametrize("rule", [Sampling(1.0, 0, 1.0), Sampling(0.8, 10, 0.9), Sampling(1.0, 0, 0.9, 0.05)])
def test_frequencies(dev, rule):
    """Tokens of evenly spread numbers come as often as they weigh: within one of n p each."""
    rng = np.random.default_rng(7)
    n, vocab = 4096, 50
    row = logits(rng, 1, vocab, "normal")[0]
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = np.bincount(_t(np.repeat(row[None], n, 0), dev).sample(u, rule).tokens(), minlength=vocab)
    ids, w, _ = keep(row, rule.temperature, rule.top_k, rule.top_p, rule.min_p)
    p = np.zeros(vocab)
    p[ids] = w / w.sum()
    assert np.all(np.abs(got - n * p) <= 1 + n * 2.0**-23)


@pytest.mark.parametrize("rows,vocab", [(1, 131072), (8, 40000), (3, 500)])
def test_captured(dev, rows, vocab):
    """On a fresh context without a workspace, and again when an eager call has made one: every replay reads the logits, numbers and
    rules that are there then."""
    rng = np.random.default_rng(8)
    hip = _hip()
    rules = [RULES[(i + 4) % len(RULES)] for i in range(rows)]
    table = np.array([[r.temperature, 0, r.top_p, r.min_p] for r in rules], np.float32)
    table.view(np.int32)[:, 1] = [r.top_k for r in rules]
    tx, tu, tr = _t(np.zeros((rows, vocab), np.float32), dev), _t(np.zeros(rows, np.float32), dev), _t(table, dev)
    to, tp = Tensor.empty([rows], dev), Tensor.empty([rows], dev)
    dev.sync()
    with _FreshCtx(dev) as f:
        call = lambda: f.lib.bch_sample(f.ctx, rows, vocab, _p(tx), vocab, None, _p(tr), _p(tu), _p(to), _p(tp))
        graphs = []
        for _ in range(2):
            assert hip.hipStreamBeginCapture(f.stream, CAPTURE_RELAXED) == 0
            st = call()
            graph, ex = C.c_void_p(), C.c_void_p()
            assert hip.hipStreamEndCapture(f.stream, C.byref(graph)) == 0 and st == 0
            assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
            graphs.append((graph, ex))
            assert call() == 0 and f.lib.bch_sync(f.ctx) == 0
        for t in range(3):
            x, u = logits(rng, rows, vocab, "peaked"), rng.random(rows, dtype=np.float32)
            dev.upload(tx.ptr, x)
            dev.upload(tu.ptr, u)
            dev.sync()
            for _, ex in graphs:
                assert hip.hipGraphLaunch(ex, f.stream) == 0 and f.lib.bch_sync(f.ctx) == 0
                assert check(x, u, rules, to.to_numpy().view(np.int32), tp.to_numpy()) == 0
            assert call() == 0 and f.lib.bch_sync(f.ctx) == 0
            assert check(x, u, rules, to.to_numpy().view(np.int32), tp.to_numpy()) == 0
        for graph, ex in graphs:
            hip.hipGraphExecDestroy(ex)
            hip.hipGraphDestroy(graph)
