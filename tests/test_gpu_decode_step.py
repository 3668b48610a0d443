"""Serving with 4-bit weights: projections, keys turned and appended, paged attention, logits and the tokens drawn from
them, as one run -- each stage against 64 bits of what the stage before it gave."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from barracuda_amd import KvCache, Rotary, Sampling, Tensor
from barracuda_amd import _native as N
from barracuda_amd.nn import Activation, Weights4, dequantize4, linear4, quantize4
from tests.kv_model import attend, visible
from tests.rotary_model import depths, turned
from tests.sample_model import choose
from tests.sample_model import slack as near_border
from tests.test_gpu_graph import CAPTURE_RELAXED, _FreshCtx, _hip
from tests.test_gpu_kv_cache import _p, _t
from tests.test_gpu_paged import compare, tolerance
from tests.test_gpu_w4 import slack

pytestmark = pytest.mark.gpu


class _Linear:
    def __init__(self, dev, rng, n, k, group, zeros=False):
        codes, scales, z = quantize4(rng.standard_normal((n, k), dtype=np.float32) / np.float32(np.sqrt(k)), group, zeros)
        self.weights = Weights4(codes, scales, k, group, z, dev)
        self.wide = dequantize4(codes, scales, group, k, z).astype(np.float64)

    def __call__(self, x, act=None):
        y = linear4(x, self.weights, None, act)
        a, got = x.to_numpy(), y.to_numpy()
        want, tol = a.astype(np.float64) @ self.wide.T, slack(a, self.wide)
        if act is Activation.GELU:  # slope at most 1.13, and its own roundings
            want = want / (1.0 + np.exp(-2.0 * 0.7978845608 * (want + 0.044715 * want**3)))
            tol = 1.13 * tol + 8 * 2.0**-24 * np.abs(want) + 1e-37
        assert np.all(np.abs(got - want) <= tol)
        return y


class _Decoder:
    """Layers of attention and a two-layer perceptron over 4-bit weights, and the model of what its cache holds."""

    def __init__(self, dev, rng, dim, h, hkv, d, page, vocab, group, zeros):
        self.dev, self.rng, self.h, self.hkv, self.d, self.vocab = dev, rng, h, hkv, d, vocab
        lin = lambda n, k: _Linear(dev, rng, n, k, group, zeros)
        self.layers = [dict(q=lin(h * d, dim), k=lin(hkv * d, dim), v=lin(hkv * d, dim), o=lin(dim, h * d),
                            up=lin(2 * dim, dim), down=lin(dim, 2 * dim)) for _ in range(2)]
        self.head = lin(vocab, dim)
        self.embed = rng.standard_normal((vocab, dim), dtype=np.float32)
        self.rotary = Rotary(d, base=500.0, device=dev)
        self.cache = KvCache(2, 64, page, hkv, d, dev)
        self.held = {}  # sequence -> per layer (keys, values), lists

    def sequence(self):
        s = self.cache.new_sequence()
        self.held[s] = [([], []) for _ in self.layers]
        return s

    def step(self, items, tokens, parents=None):
        """The logits of every new token."""
        step = self.cache.batch(items, parents)
        x = _t(self.embed[np.asarray(tokens)], self.dev)
        row = lambda i: slice(int(step.start[i]), int(step.start[i + 1]))
        for at, layer in enumerate(self.layers):
            q, k, v = (layer[n](x).reshape([step.total, heads, self.d])
                       for n, heads in (("q", self.h), ("k", self.hkv), ("v", self.hkv)))
            tq = self.cache.append_rotary(step, at, self.rotary, q, k, v)
            y = self.cache.attention(step, at, tq)
            q, k, v, tq_, y_ = (t.to_numpy() for t in (q, k, v, tq, y))
            for i, (s, n) in enumerate(items):
                if n == 0:
                    continue
                r = row(i)
                first = len(self.held[s][at][0])
                where = first + (np.array(depths(parents[i])) if parents else np.arange(n))
                want, tol = turned(q[r], where[:, None], self.rotary.freqs, self.d, False, 1.0)
                assert np.all(np.abs(tq_[r] - want) <= tol)
                keys, values = self.held[s][at]
                # the keys as they would be at best; rounding them to 32 bits moves each by less than its own tolerance
                keys.extend(turned(k[r], where[:, None], self.rotary.freqs, self.d, False, 1.0)[0].astype(np.float32))
                values.extend(v[r])
                scale = float(np.float32(1.0) / np.sqrt(np.float32(self.d)))
                ks, vs = np.stack(keys), np.stack(values)
                want = attend(tq_[r], ks, vs, visible(first, n, 0, 0, parents[i] if parents else None), scale)
                # a key's columns are off by 5 * 2^-24 of a pair's two magnitudes, which sum to at most sqrt(2) of their length: a
                # score by that of the lengths' product, a weighted mean by twice as much (numerator and denominator)
                s_max = scale * np.sqrt((tq_[r].astype(np.float64) ** 2).sum(-1).max() * (ks.astype(np.float64) ** 2).sum(-1).max())
                compare(y_[r], want, tolerance(tq_[r], ks, vs, scale, len(keys)) + 2 * 2 * 5 * 2.0**-24 * s_max * np.abs(vs).max())
            x = layer["o"](y.reshape([step.total, self.h * self.d]))
            x = layer["down"](layer["up"](x, Activation.GELU))
        return step, self.head(x)

    def draw(self, logits, rules):
        rows = logits.shape()[0]
        u = self.rng.random(rows, dtype=np.float32)
        out = logits.sample(u, rules)
        got, x = out.tokens(), logits.to_numpy()
        for i in range(rows):
            t = rules[i].temperature
            token, prob, near = choose(x[i], u[i], t, rules[i].top_k, rules[i].top_p, rules[i].min_p)
            if near > near_border(x[i], t):
                assert got[i] == token
        assert np.all((got >= 0) & (got < self.vocab))
        return got

    def last(self, step, logits):
        """The logits of each sequence's last new token, as rows of their own."""
        return _t(logits.to_numpy()[step.start[1:] - 1], self.dev)


@pytest.mark.parametrize("dim,h,hkv,d,page,vocab,group,zeros", [(192, 6, 2, 64, 16, 1000, 64, False),
                                                                (160, 3, 3, 80, 5, 20001, 32, True)])
def test_prompts_tokens_and_drafts(dev, dim, h, hkv, d, page, vocab, group, zeros):
    rng = np.random.default_rng(d)
    m = _Decoder(dev, rng, dim, h, hkv, d, page, vocab, group, zeros)
    a, b, c = (m.sequence() for _ in range(3))
    rules = [Sampling(0.8, 40, 0.95), Sampling(0.0), Sampling(1.2, 0, 0.9, 0.01)]
    step, logits = m.step([(a, 37), (b, 1), (c, 90)], rng.integers(0, vocab, 128))
    tokens = m.draw(m.last(step, logits), rules)
    for _ in range(3):
        _, logits = m.step([(a, 1), (b, 1), (c, 1)], tokens)
        tokens = m.draw(logits, rules)
    # drafts of two sequences; the ones that are kept close up, the third sequence had none
    parents = [[-1, 0, 0, 1], [], [-1, -1, 1]]
    step, logits = m.step([(a, 4), (b, 0), (c, 3)], np.concatenate([tokens[:1], rng.integers(0, vocab, 3), tokens[2:], [1, 2]]),
                          parents)
    m.draw(logits, [rules[0]] * 4 + [rules[2]] * 3)
    m.cache.keep(step, [[0, 1, 3], [], [1, 2]])
    for s, n, ids in ((a, 4, [0, 1, 3]), (c, 3, [1, 2])):
        for keys, values in m.held[s]:
            for held in (keys, values):
                old = len(held) - n
                held[:] = held[:old] + [held[old + i] for i in ids]
    _, logits = m.step([(c, 1), (a, 1), (b, 1)], tokens[[2, 0, 1]])
    m.draw(logits, rules)


@pytest.mark.parametrize("rows,dim,h,hkv,d,vocab", [(1, 256, 4, 2, 64, 50021), (5, 256, 4, 2, 64, 2000), (24, 512, 8, 2, 64, 20000)])
def test_captured_token(dev, rows, dim, h, hkv, d, vocab):
    """One token of every sequence as a graph, from projections to the draw: replayed with other inputs, lengths and numbers it
    gives what the calls give one by one, with the program's own calls on the same workspace between the replays."""
    rng = np.random.default_rng(rows)
    page, width = 16, 8
    lin = lambda n, k: Weights4.quantize(rng.standard_normal((n, k), dtype=np.float32) / np.float32(np.sqrt(k)), 64, device=dev)
    wq, wk, wv, wo, head = lin(h * d, dim), lin(hkv * d, dim), lin(hkv * d, dim), lin(dim, h * d), lin(vocab, dim)
    pool = rng.standard_normal((2, rows * width, hkv, page, d), dtype=np.float32)
    x, u = Tensor.empty([rows, dim], dev), Tensor.empty([rows], dev)
    q, k, v = (Tensor.empty([rows, n, d], dev) for n in (h, hkv, hkv))
    y, o, logits, probs = (Tensor.empty(s, dev) for s in ([rows, h * d], [rows, dim], [rows, vocab], [rows]))
    tokens, lengths = Tensor.empty([rows], dev), Tensor.empty([rows], dev)
    keys, values = _t(pool[0], dev), _t(pool[1], dev)
    start, table = Tensor.empty([rows + 1], dev), Tensor.empty([rows, width], dev)
    dev.upload(start.ptr, np.arange(rows + 1, dtype=np.int32))
    dev.upload(table.ptr, rng.permutation(rows * width).astype(np.int32))
    lay = N.AttnLayout(hkv * page * d, page * d, d)
    pages = N.KvPages(keys.ptr, values.ptr, lay, lay, rows * width, page, hkv, d, table.ptr, width)
    batch = N.KvBatch(rows, rows, 1, page * width, start.ptr, lengths.ptr)
    rotary = Rotary(d, device=dev)
    row = lambda n: N.AttnLayout(0, d, n * d)
    rule = N.Sampling(0.9, 50, 0.95, 0.0)
    dev.sync()
    with _FreshCtx(dev) as f:
        lib = f.lib
        linear = lambda a, w, n, kk, c: lib.bch_w4_linear(f.ctx, rows, w._w, _p(a), kk, None, N.BCH_ACT_NONE, _p(c), n)

        def call():
            return [linear(x, wq, h * d, dim, q), linear(x, wk, hkv * d, dim, k), linear(x, wv, hkv * d, dim, v),
                    lib.bch_kv_append_rotary(f.ctx, pages, batch, None, rotary._plan, h, _p(q), row(h), _p(q), row(h), _p(k), row(hkv),
                                             _p(v), row(hkv)),
                    lib.bch_sdpa_paged(f.ctx, pages, batch, h, d**-0.5, 0, 0, None, _p(q), row(h), _p(y), row(h)),
                    linear(y, wo, dim, h * d, o), linear(o, head, vocab, dim, logits),
                    lib.bch_sample(f.ctx, rows, vocab, _p(logits), vocab, rule, None, _p(u), _p(tokens), _p(probs))]

        def give(seed):
            r = np.random.default_rng(seed)
            for t, a in ((x, r.standard_normal((rows, dim), dtype=np.float32)), (u, r.random(rows, dtype=np.float32)),
                         (lengths, r.integers(1, page * width + 1, rows).astype(np.int32)), (keys, pool[0]), (values, pool[1])):
                dev.upload(t.ptr, a)
            dev.sync()

        def results():
            assert lib.bch_sync(f.ctx) == 0
            return [t.to_numpy().copy() for t in (q, keys, values, y, logits, tokens, probs)]

        give(0)
        assert not any(call())  # sizes the workspace
        results()
        hip, graph, ex = _hip(), C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(f.stream, CAPTURE_RELAXED) == 0
        st = call()
        assert hip.hipStreamEndCapture(f.stream, C.byref(graph)) == 0 and not any(st)
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
        for seed in range(1, 5):
            give(seed)
            assert not any(call())
            want = results()
            give(seed)
            for t in (y, logits, tokens, probs):
                dev.upload(t.ptr, np.full(t.len(), np.nan, np.float32))
            dev.sync()
            assert hip.hipGraphLaunch(ex, f.stream) == 0
            for a, b in zip(results(), want):
                assert np.array_equal(a.view(np.int32), b.view(np.int32))
            for i in range(rows):
                token, _, near = choose(want[4][i], u.to_numpy()[i], 0.9, 50, 0.95, 0.0)
                assert near <= near_border(want[4][i], 0.9) or want[5].view(np.int32)[i] == token
        hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(graph)


def test_two_contexts_at_once(dev):
    """Calls of two contexts, one behind the other without a wait: each has its own stream and scratch, and gives what it gives alone."""
    rng = np.random.default_rng(77)
    rows, k, n = 20, 1024, 30011
    w = Weights4.quantize(rng.standard_normal((n, k), dtype=np.float32), 64, device=dev)
    xs = [_t(rng.standard_normal((rows, k), dtype=np.float32), dev) for _ in range(2)]
    us = [_t(rng.random(rows, dtype=np.float32), dev) for _ in range(2)]
    out = [(Tensor.empty([rows, n], dev), Tensor.empty([rows], dev), Tensor.empty([rows], dev)) for _ in range(2)]
    rules = [N.Sampling(1.0, 0, 0.9, 0.0), N.Sampling(0.7, 30, 0.95, 0.0)]
    dev.sync()
    with _FreshCtx(dev) as f, _FreshCtx(dev) as g:
        def call(c, i):
            y, tokens, probs = out[i]
            assert c.lib.bch_w4_linear(c.ctx, rows, w._w, _p(xs[i]), k, None, N.BCH_ACT_NONE, _p(y), n) == 0
            assert c.lib.bch_sample(c.ctx, rows, n, _p(y), n, rules[i], None, _p(us[i]), _p(tokens), _p(probs)) == 0

        def results():
            assert f.lib.bch_sync(f.ctx) == 0 and g.lib.bch_sync(g.ctx) == 0
            return [t.to_numpy().view(np.int32).copy() for o in out for t in o]

        call(f, 0)
        alone = results()[:3]
        call(g, 1)
        alone += results()[3:]
        for _ in range(3):
            for _ in range(10):
                call(f, 0)
                call(g, 1)
            for a, b in zip(results(), alone):
                assert np.array_equal(a, b)
