"""Sampling gives a token by the logits, the rule and the number alone, on the GPU: with and without a workspace, whichever kernels
take a row."""
from __future__ import annotations

import numpy as np
import pytest

from barracuda_amd import Sampling, Tensor
from tests.sample_model import choose, slack
from tests.test_gpu_graph import _FreshCtx
from tests.test_gpu_kv_cache import _p, _t
from tests.test_gpu_sample import MANY, RULES, logits

pytestmark = pytest.mark.gpu


def table(rules):
    """Rules as they lie in device memory."""
    t = np.array([[r.temperature, 0, r.top_p, r.min_p] for r in rules], np.float32)
    t.view(np.int32)[:, 1] = [min(int(r.top_k), 2**31 - 1) for r in rules]
    return t


def both(dev, monkeypatch, x, u, rules):
    """(tokens, probabilities) of a context that has a workspace, and of one that gets none."""
    rows, vocab = x.shape
    tx, tu, tr = _t(x, dev), _t(u, dev), _t(table(rules), dev)
    to, tp = Tensor.empty([rows], dev), Tensor.empty([rows], dev)
    dev.sync()
    out = []
    for fail in ("0", "1"):
        with _FreshCtx(dev) as f:
            monkeypatch.setenv("BARRACUDA_HIP_FAIL_WORKSPACE", fail)
            assert f.lib.bch_sample(f.ctx, rows, vocab, _p(tx), vocab, None, _p(tr), _p(tu), _p(to), _p(tp)) == 0
            assert f.lib.bch_sync(f.ctx) == 0
            out.append((to.to_numpy().view(np.int32).copy(), tp.to_numpy().copy()))
    monkeypatch.delenv("BARRACUDA_HIP_FAIL_WORKSPACE")
    return out


def units_log(vocab):
    bits = 1
    while (1 << bits) <= vocab:
        bits += 1
    return min(51, 62 - bits)


def test_many_light_tokens_without_a_cut(dev, monkeypatch):
    """All but the last token weigh 2^-46 of it, half of what whole numbers of 2^-44 hold: together 2^-29 of the whole, which a
    number of 2^-31 falls into.  The same with the heavy token in the middle."""
    vocab = 131072
    x = np.full((4, vocab), -46 * np.log(2), np.float32)
    x[:2, -1] = x[2:, 70000] = 0
    u = np.array([2.0**-31, 2.0**-28, 2.0**-32, 1 - 2.0**-24], np.float32)
    (a, pa), (b, pb) = both(dev, monkeypatch, x, u, [Sampling()] * 4)
    light = np.exp(np.float64(x[0, 0]))
    assert np.array_equal(a, [int(2.0**-31 * (1 + light * (vocab - 1)) / light), vocab - 1,
                              int(2.0**-32 * (1 + light * (vocab - 1)) / light), 70000])
    assert np.array_equal(a, b) and np.array_equal(pa, pb)


def border_row(rng, vocab):
    """A row whose light tokens' weights are rounded down by 0.4 to 0.5 units each, and (top_p, tokens) so that what top_p asks for
    ends between the heavy tokens' weights with the whole from rounded weights and with the whole as it is."""
    unit = 2.0 ** units_log(vocab)
    light = rng.uniform(-16, -12, vocab - 200).astype(np.float32)
    tries = light[:, None] * (1 + np.arange(48, dtype=np.float32) * np.float32(2.0**-23))
    part = np.exp(tries.astype(np.float64)) * unit % 1.0
    at = np.argmin(np.abs(part - 0.47), 1)
    light, part = np.take_along_axis(tries, at[:, None], 1)[:, 0], np.take_along_axis(part, at[:, None], 1)[:, 0]
    heavy = np.sort(rng.uniform(-9, -5, 200).astype(np.float32))[::-1]
    heavy[0] = 0
    heavy_units = np.rint(np.exp(heavy.astype(np.float64)) * unit)
    rounded = heavy_units.sum() + np.rint(np.exp(light.astype(np.float64)) * unit).sum()
    real = heavy_units.sum() + (np.exp(light.astype(np.float64)) * unit).sum()
    margin = 2000.0  # units; what weights of 2^-51 of their span's largest and sums in 64 bits leave open is less
    found = []
    for n in range(20, 150):
        run = heavy_units[:n].sum()
        p = np.float32((run / rounded + run / real) / 2)
        if float(p) * real > run + margin and float(p) * rounded < run - margin:
            found.append((p, n + 1))
    x = np.empty(vocab, np.float32)
    where = rng.permutation(vocab)
    x[np.sort(where[:200])] = heavy  # in index order, so that the last that is left is the lightest
    x[where[200:]] = light
    return x, found, np.sort(where[:200])


def test_a_border_between_two_sums_of_the_row(dev, monkeypatch):
    """The whole that top_p cuts a part of is one sum, whichever kernels take the row."""
    rng = np.random.default_rng(1)
    vocab, rows, rules, want = 131072, [], [], []
    for _ in range(12):
        x, found, where = border_row(rng, vocab)
        for p, n in found:
            rows.append(x)
            rules.append(Sampling(1.0, 0, float(p)))
            want.append(where[n - 1])
    assert len(rows) >= 12
    u = np.full(len(rows), 1 - 2.0**-24, np.float32)
    (a, pa), (b, pb) = both(dev, monkeypatch, np.stack(rows), u, rules)
    assert np.array_equal(a, want)
    assert np.array_equal(b, want) and np.array_equal(pa, pb)


@pytest.mark.parametrize("kind", ["normal", "peaked", "flat", "coarse", "equal", "masked", "wide"])
@pytest.mark.parametrize("vocab", [8193, 20011, 131072])
def test_rules_with_and_without_a_workspace(dev, monkeypatch, vocab, kind):
    rng = np.random.default_rng(vocab + 1)
    rules = RULES + MANY
    x, u = logits(rng, len(rules), vocab, kind), rng.random(len(rules), dtype=np.float32)
    (a, pa), (b, pb) = both(dev, monkeypatch, x, u, rules)
    assert np.array_equal(a, b) and np.array_equal(pa, pb)
    for i, r in enumerate(rules):
        token, _, near = choose(x[i], u[i], r.temperature, r.top_k, r.top_p, r.min_p)
        assert a[i] == token or near <= slack(x[i], r.temperature)


@pytest.mark.parametrize("mask", [-1e9, -65504.0, np.finfo(np.float32).min])
@pytest.mark.parametrize("vocab,n", [(600, 5), (9000, 40), (50021, 300), (50021, 5000)])
def test_masks_of_finite_numbers(dev, monkeypatch, vocab, n, mask):
    """A mask by a type's lowest number instead of -inf: masked tokens weigh nothing, but a top_k beyond the others takes them in."""
    rng = np.random.default_rng(n)
    rules = RULES + MANY
    x = np.full((len(rules), vocab), mask, np.float32)
    for r in x:
        r[rng.permutation(vocab)[:n]] = 2 * rng.standard_normal(n, dtype=np.float32)
    u = rng.random(len(rules), dtype=np.float32)
    (a, pa), (b, pb) = both(dev, monkeypatch, x, u, rules)
    assert np.array_equal(a, b) and np.array_equal(pa, pb)
    for i, r in enumerate(rules):
        token, p, near = choose(x[i], u[i], r.temperature, r.top_k, r.top_p, r.min_p)
        if near > slack(x[i], r.temperature):
            assert a[i] == token and abs(pa[i] - p) <= 2.0**-24 * p + 2 * slack(x[i], r.temperature), (i, r)
