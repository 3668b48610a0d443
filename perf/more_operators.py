"""Timed cases of what a decode step does around its attention: rotary positions, linear layers of 4-bit weights, sampling.

Each case is one pass through an operator as a serving program makes it:

  rotary   queries or keys of a dense tensor turned by their positions, or turned    bch_rotary
           back (the gradient of the turn)
  append   new tokens' q turned, their k turned and stored with v in the pages of    bch_kv_append_rotary
           a paged cache; a chunk of a prompt, one token a sequence, or drafted trees
  w4       a linear layer with 4-bit weights, a scale and a zero point for each      bch_w4_linear
           group of inputs
  sample   a token for each row of logits, from given numbers                        bch_sample

Rotary: columns i and i + dim/2 of a head (interleaved: 2i and 2i + 1) are turned by position * freq[i] and multiplied by
`scale`; columns from dim on stay.  New token i of a sequence with len keys, n of them new, stands at position len - n + i; a
drafted one behind its parent.

w4: y = act(x W^T + bias), W[o][i] = scales[o][i / group] * (code[o][i] - zero[o][i / group]), two codes a byte.

sample: with w_i = exp((x_i - max) / temperature), of the top_k largest logits (ties: the lower index first), of these the
shortest beginning that holds top_p of their weight, of these the ones with w_i >= min_p, the first in index order whose
cumulative weight exceeds u times the whole.  Temperature 0 takes the largest logit.  A row of nothing but -inf gives -1.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # queries of a batch of prompts, bench.py's attention shape
        {"name": "rotary_dense", "kind": "rotary", "b": 4, "h": 32, "s": 2048, "d": 128, "dim": 128, "interleaved": False,
         "heads_last": False, "back": False, "scaling": "none", "far": 0},
        # gradients turned back in a projection's own layout, an odd length, part of the head, a long-context scaling
        {"name": "rotary_back", "kind": "rotary", "b": 3, "h": 12, "s": 1023, "d": 80, "dim": 40, "interleaved": True,
         "heads_last": True, "back": True, "scaling": "parts", "far": 100000},
        # the decode step of 32 conversations: launch latency counts
        {"name": "append_decode", "kind": "append", "b": 32, "h": 32, "hkv": 8, "d": 128, "dim": 128, "interleaved": False,
         "scaling": "none", "len": 1024, "new": 1, "page": 16, "ragged": True, "tree": False},
        # prompts of different lengths
        {"name": "append_prefill", "kind": "append", "b": 8, "h": 32, "hkv": 8, "d": 128, "dim": 128, "interleaved": False,
         "scaling": "linear", "len": 4096, "new": 4096, "page": 64, "ragged": True, "tree": False},
        # a verification step: trees of 64 drafts, half of each head turned
        {"name": "append_tree", "kind": "append", "b": 16, "h": 16, "hkv": 4, "d": 64, "dim": 32, "interleaved": True,
         "scaling": "none", "len": 700, "new": 64, "page": 16, "ragged": True, "tree": True},
        # one conversation's token through a projection of bench.py's decode shape
        {"name": "w4_decode_one", "kind": "w4", "m": 1, "k": 4096, "n": 11008, "group": 128, "zeros": False, "bias": False,
         "act": "none"},
        # a decode step of 32 conversations, the way back of the same block
        {"name": "w4_decode_batch", "kind": "w4", "m": 32, "k": 11008, "n": 4096, "group": 128, "zeros": True, "bias": True,
         "act": "none"},
        # a narrow odd layer with small groups
        {"name": "w4_ragged", "kind": "w4", "m": 7, "k": 1001, "n": 2999, "group": 32, "zeros": True, "bias": True,
         "act": "gelu"},
        # a prompt's tokens: the largest case
        {"name": "w4_prompt", "kind": "w4", "m": 2048, "k": 4096, "n": 11008, "group": 128, "zeros": False, "bias": True,
         "act": "gelu"},
        # one conversation's next token
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 32768, "temperature": 0.8, "top_k": 40, "top_p": 0.95,
         "min_p": 0.0, "mixed": False, "masked": False},
        # the next tokens of a large batch, each conversation with its own settings
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 131072, "temperature": 1.0, "top_k": 50, "top_p": 0.9,
         "min_p": 0.02, "mixed": True, "masked": False},
        # rows that a grammar leaves few tokens of, one none, at a high temperature
        {"name": "sample_masked", "kind": "sample", "rows": 16, "vocab": 50021, "temperature": 1.3, "top_k": 0, "top_p": 0.98,
         "min_p": 0.0, "mixed": False, "masked": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of them."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 1.84e11 and w["bytes"] <= 4.9e8 and _pool_floats(case) <= 3.4e7:
            return case


def _draw(rng):
    kind = rng.choice(["rotary", "append", "append", "w4", "w4", "w4", "sample", "sample"])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 200, 256])
    turn = {"d": d, "dim": rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]), "interleaved": rng.random() < 0.4,
            "scaling": rng.choice(["none", "none", "linear", "base", "parts"])}
    if kind == "rotary":
        return {"kind": kind, "b": rng.randint(1, 8), "h": rng.randint(1, 40), "s": _log(rng, 1, 4096), **turn,
                "heads_last": rng.random() < 0.5, "back": rng.random() < 0.5, "far": rng.choice([0, 0, 1000, 100000, 1 << 22])}
    if kind == "append":
        hkv = rng.choice([1, 2, 4, 8])
        tree = rng.random() < 0.3
        length = _log(rng, 2, 8192)
        new = _log(rng, 1, min(length, 128)) if tree else 1 if rng.random() < 0.4 else _log(rng, 1, length)
        return {"kind": kind, "b": _log(rng, 1, 48), "h": hkv * rng.choice([1, 2, 4, 8]), "hkv": hkv, **turn, "len": length,
                "new": new, "page": rng.choice([1, 8, 16, 16, 24, 64, 64, 128]), "ragged": rng.random() < 0.7, "tree": tree}
    if kind == "w4":
        m = rng.choice([1, 1, 2, 4, 8]) if rng.random() < 0.4 else _log(rng, 1, 2048)
        return {"kind": kind, "m": m, "k": _log(rng, 64, 12288), "n": _log(rng, 64, 12288),
                "group": rng.choice([32, 64, 128, 128, 256]), "zeros": rng.random() < 0.5, "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "none", "relu", "gelu"])}
    return {"kind": kind, "rows": _log(rng, 1, 128), "vocab": _log(rng, 500, 200000),
            "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]), "top_k": rng.choice([0, 0, 1, _log(rng, 2, 2000)]),
            "top_p": rng.choice([1.0, 1.0, 0.98, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
            "mixed": rng.random() < 0.4, "masked": rng.random() < 0.3}


# ---- what a case's sequences are ------------------------------------------------------


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _sequences(case):
    """Keys and new tokens of every sequence: the first one's are the case's, ragged ones' are anything up to it."""
    r = _rng(case)
    lens, news = [case["len"]], [case["new"]]
    for b in range(1, case["b"]):
        if not case["ragged"]:
            lens.append(lens[0])
            news.append(news[0])
            continue
        new = 1 if case["new"] == 1 else 0 if b == 3 else _log(r, 1, case["new"])
        lens.append(max(new, _log(r, 1, case["len"])))
        news.append(new)
    return lens, news


def _parents(case):
    """For each sequence its drafts' parents, -1 for a child of the last committed token."""
    r = _rng(case)
    return [[-1 if i == 0 or r.random() < 0.1 else r.randint(max(0, i - 8), i - 1) for i in range(n)]
            for n in _sequences(case)[1]]


def _pool_floats(case):
    if case["kind"] != "append":
        return 0
    pages = sum(-(-length // case["page"]) for length in _sequences(case)[0])
    return pages * case["page"] * case["hkv"] * case["d"]


def _rules(case):
    """Temperature, top_k, top_p and min_p of every row."""
    one = (case["temperature"], case["top_k"], case["top_p"], case["min_p"])
    if not case["mixed"]:
        return [one] * case["rows"]
    r = _rng(case)
    others = [one, (0.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 20, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 200, 0.95, 0.01),
              (1.0, 0, 1.0, 0.0)]
    return [one if i == 0 else r.choice(others) for i in range(case["rows"])]


def _freq(case):
    """Radians a position for each pair of columns, in 64 bits."""
    dim, scaling = case["dim"], case["scaling"]
    base, factor, first_context = 10000.0, 4.0, 8192.0
    if scaling == "base" and dim > 2:  # the slowest pair is slowed by the factor, the fastest not at all
        base *= factor ** (dim / (dim - 2.0))
    f = base ** (-2.0 * np.arange(dim // 2) / dim)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":  # pairs that turn more than 32 times in the first context stay, those below once are slowed
        stay = np.clip((first_context * f / (2.0 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        f = f * (stay + (1.0 - stay) / factor)
    return f


def _turn_scale(case):
    return 0.1 * math.log(4.0) + 1.0 if case["scaling"] == "parts" else 1.0


# ---- inputs ---------------------------------------------------------------------------


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda").reshape(-1)


def _inputs(case, seed):
    """The case's inputs as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind == "rotary":
        b, h, s, d = (case[x] for x in "bhsd")
        x = {"x": normal(b, s, h, d) if case["heads_last"] else normal(b, h, s, d)}
        if case["far"]:  # each row's position is given: contiguous from some far place on
            first = torch.randint(0, case["far"], (b, 1), generator=g, device="cuda")
            x["positions"] = (first + torch.arange(s, device="cuda")).to(torch.int32)
        x["freq"] = torch.from_numpy(_freq(case)).cuda()
        return x
    if kind == "append":
        hkv, d, page = case["hkv"], case["d"], case["page"]
        lens, news = _sequences(case)
        held = [-(-length // page) for length in lens]
        pages = sum(held) + max(1, sum(held) // 16)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(held):
            table[b, :n] = order[at:at + n]
            at += n
        start = np.concatenate([[0], np.cumsum(news)]).tolist()
        total = start[-1]
        x = {"table": table, "len": _i32(lens), "start": _i32(start), "q": normal(total, case["h"], d),
             "new_k": normal(total, hkv, d), "new_v": normal(total, hkv, d), "freq": torch.from_numpy(_freq(case)).cuda()}
        if case["tree"]:
            x["parent"] = _i32([p for seq in _parents(case) for p in seq])
        # pools as the cache lays them out: a head's keys of a page side by side
        x["k"], x["v"] = normal(pages, hkv, page, d), normal(pages, hkv, page, d)
        return x
    if kind == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        x = {"x": normal(m, k),
             "codes": torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8),
             "scale": (0.5 + torch.rand(n, groups, generator=g, device="cuda")) * (0.3 / math.sqrt(k))}
        if case["zeros"]:
            x["zero"] = torch.randint(4, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
        if case["bias"]:
            x["bias"] = normal(n)
        return x
    rows, vocab = case["rows"], case["vocab"]
    # most logits in a bell, a few far above it
    logits = 2.0 * normal(rows, vocab)
    tall = torch.rand(rows, vocab, generator=g, device="cuda") < 1e-3
    logits += tall * -2.5 * torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_min(1e-6))
    if case["masked"]:
        logits.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < 0.9, -math.inf)
        if rows > 3:
            logits[3] = -math.inf
    rules = np.zeros((rows, 4), dtype=np.float32)
    rules[:] = _rules(case)
    whole = rules.view(np.int32).copy()
    whole[:, 1] = rules[:, 1].astype(np.int32)
    return {"logits": logits, "u": torch.rand(rows, generator=g, device="cuda"), "rules": torch.from_numpy(whole).cuda()}


def _p(x):
    return ctypes.c_void_p(x.data_ptr()) if x is not None else None


def _handles(case, x):
    """What a serving program keeps beside its buffers: the plan of the turn, the cache's description and the step's batch,
    the weights in the layout that the kernels read, and the buffers that results go to."""
    from barracuda_amd import _native, get_device
    dev, lib = get_device(), _native.load()
    s = {"dev": dev, "lib": lib}
    kind = case["kind"]
    torch.cuda.synchronize()
    if kind in ("rotary", "append"):
        s["turn"] = _native.Rotary(case["dim"], int(case["interleaved"]), _turn_scale(case), x["freq"].data_ptr())
    if kind == "rotary":
        h, n, d = (case[i] for i in "hsd")
        s["layout"] = _native.AttnLayout(h * n * d, d, h * d) if case["heads_last"] else _native.AttnLayout(h * n * d, n * d, d)
        s["o"] = torch.empty_like(x["x"])
    elif kind == "append":
        pages, hkv, page, d = x["k"].shape
        layout = _native.AttnLayout(hkv * page * d, page * d, d)
        lens, news = _sequences(case)
        s["kv"] = _native.KvPages(x["k"].data_ptr(), x["v"].data_ptr(), layout, layout, pages, page, hkv, d,
                                  x["table"].data_ptr(), x["table"].shape[1])
        s["batch"] = _native.KvBatch(len(lens), sum(news), max(news), max(lens), x["start"].data_ptr(), x["len"].data_ptr())
        s["q_rows"], s["kv_rows"] = _native.AttnLayout(0, d, case["h"] * d), _native.AttnLayout(0, d, hkv * d)
        s["o"] = torch.empty_like(x["q"])
    elif kind == "w4":
        n, k = case["n"], case["k"]
        size = ctypes.c_size_t()
        dev.check(lib.bch_w4_bytes(n, k, case["group"], ctypes.byref(size)), "w4_bytes")
        s["packed"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        dev.check(lib.bch_w4_pack(dev.ctx, n, k, case["group"], _p(x["codes"]), x["codes"].shape[1], _p(x["scale"]),
                                  _p(x.get("zero")), _p(s["packed"])), "w4_pack")
        s["w"] = _native.W4(n, k, case["group"], s["packed"].data_ptr())
        s["act"] = {"none": _native.BCH_ACT_NONE, "relu": _native.BCH_ACT_RELU, "gelu": _native.BCH_ACT_GELU}[case["act"]]
        s["y"] = torch.empty(case["m"], n, device="cuda")
        dev.sync()
    else:
        rows = case["rows"]
        s["one"] = _native.Sampling(case["temperature"], case["top_k"], case["top_p"], case["min_p"])
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["probs"] = torch.empty(rows, device="cuda")
    return s


def prepare(case, seed):
    """Inputs, weights, cache, tables and handles in HBM; the outputs that a serving loop holds."""
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if own:
        state.update(_handles(case, x))
    torch.cuda.synchronize()
    return state


# ---- one pass ---------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state["case"], state["x"])


def _run_own(s):
    case, x, dev, lib = s["case"], s["x"], s["dev"], s["lib"]
    kind = case["kind"]
    if kind == "rotary":
        dev.check(lib.bch_rotary(dev.ctx, case["b"], case["h"], case["s"], case["d"], s["turn"], int(case["back"]), 0,
                                 _p(x.get("positions")), _p(x["x"]), s["layout"], _p(s["o"]), s["layout"]), "rotary")
        return s["o"]
    if kind == "append":
        dev.check(lib.bch_kv_append_rotary(dev.ctx, s["kv"], s["batch"], _p(x.get("parent")), s["turn"], case["h"], _p(x["q"]),
                                           s["q_rows"], _p(s["o"]), s["q_rows"], _p(x["new_k"]), s["kv_rows"],
                                           _p(x["new_v"]), s["kv_rows"]), "append")
        return [s["o"], x["k"], x["v"]]
    if kind == "w4":
        dev.check(lib.bch_w4_linear(dev.ctx, case["m"], s["w"], _p(x["x"]), case["k"], _p(x.get("bias")), s["act"], _p(s["y"]),
                                    case["n"]), "linear4")
        return s["y"]
    dev.check(lib.bch_sample(dev.ctx, case["rows"], case["vocab"], _p(x["logits"]), case["vocab"], s["one"],
                             _p(x["rules"]) if case["mixed"] else None, _p(x["u"]), _p(s["tokens"]), _p(s["probs"])), "sample")
    return [s["tokens"], s["probs"]]


# the plain form: 32 bits, but for angles and the weights that a choice hangs on


def _turned(x, angle, case):
    """x [..., D] turned by angle [..., dim / 2] (float64)."""
    dim, scale = case["dim"], _turn_scale(case)
    c, s = (scale * torch.cos(angle)).float(), (scale * torch.sin(angle)).float()
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:dim:2], x[..., 1:dim:2]
        out[..., 0:dim:2], out[..., 1:dim:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :dim // 2], x[..., dim // 2:dim]
        out[..., :dim // 2], out[..., dim // 2:dim] = a * c - b * s, a * s + b * c
    return out


def _depth(parent, start, total):
    """Of each draft the number of its ancestors, all sequences together: each step joins a draft's ancestors with those of the
    furthest one."""
    which = torch.repeat_interleave(torch.arange(start.shape[0] - 1, device="cuda"), start[1:] - start[:-1], output_size=total)
    # row `total` stands for the committed tokens
    at = torch.full((total + 1,), total, device="cuda")
    at[:total] = torch.where(parent >= 0, parent.long() + start[which], total)
    depth = (at < total).long()
    for _ in range(7):  # at most 128 drafts
        depth += depth[at]
        at = at[at]
    return depth[:total]


def _weights(case, x):
    """The 4-bit weights as float32, [n, k]."""
    n, k, group = case["n"], case["k"], case["group"]
    code = torch.stack([x["codes"] & 15, x["codes"] >> 4], 2).view(n, -1)[:, :k].float()
    pick = torch.arange(k, device="cuda") // group
    zero = x["zero"].float()[:, pick] if "zero" in x else 8.0
    return (code - zero) * x["scale"][:, pick]


def _run_plain(case, x):
    kind = case["kind"]
    if kind == "rotary":
        b, s = case["b"], case["s"]
        pos = x["positions"].double() if "positions" in x else torch.arange(s, dtype=torch.float64, device="cuda").expand(b, s)
        angle = pos[:, :, None] * x["freq"] * (-1.0 if case["back"] else 1.0)
        return _turned(x["x"], angle[:, :, None] if case["heads_last"] else angle[:, None], case)
    if kind == "append":
        start = x["start"].long()
        n = start[1:] - start[:-1]
        total = x["q"].shape[0]
        which = torch.repeat_interleave(torch.arange(n.shape[0], device="cuda"), n, output_size=total)
        slot = (x["len"].long() - n - start[:-1])[which] + torch.arange(total, device="cuda")
        pos = (x["len"].long() - n)[which] + _depth(x["parent"], start, total) if case["tree"] else slot
        angle = (pos.double()[:, None] * x["freq"])[:, None]
        page, at = x["table"][which, slot // case["page"]].long(), slot % case["page"]
        x["k"][page, :, at] = _turned(x["new_k"], angle, case)
        x["v"][page, :, at] = x["new_v"]
        return [_turned(x["q"], angle, case), x["k"], x["v"]]
    if kind == "w4":
        y = torch.matmul(x["x"], _weights(case, x).t())
        if case["bias"]:
            y = y + x["bias"]
        if case["act"] == "relu":
            y = torch.maximum(y, torch.zeros_like(y))
        if case["act"] == "gelu":
            y = 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
        return y
    logits, rules = x["logits"], x["rules"]
    rows, vocab = logits.shape
    real = rules.view(torch.float32).double()
    temperature, top_k, top_p, min_p = real[:, :1], rules[:, 1:2].long(), real[:, 2:3], real[:, 3:4]
    greedy = temperature <= 0
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)
    top = value[:, :1].double()
    w = torch.exp((value.double() - top) / torch.where(greedy, torch.ones_like(temperature), temperature))
    w = torch.where(value == -math.inf, torch.zeros_like(w), w)
    rank = torch.arange(vocab, device="cuda")
    keep = torch.where(greedy, rank < 1, (top_k <= 0) | (rank < top_k))
    w = torch.where(keep, w, torch.zeros_like(w))
    run_sum = torch.cumsum(w, 1)
    keep = keep & ((top_p >= 1) | (rank < 1) | (run_sum - w < top_p * run_sum[:, -1:])) & (w >= min_p)
    w = torch.where(keep, w, torch.zeros_like(w))
    spread = torch.zeros_like(w).scatter_(1, order, w)
    run_sum = torch.cumsum(spread, 1)
    token = (run_sum <= x["u"].double()[:, None] * run_sum[:, -1:]).sum(1, keepdim=True)
    last = torch.where(spread > 0, rank, torch.zeros_like(rank)).amax(1, keepdim=True)
    token = torch.minimum(token, last)
    empty = top == -math.inf
    prob = spread.gather(1, token) / run_sum[:, -1:]
    return [torch.where(empty, -1, token).view(-1).to(torch.int32),
            torch.where(empty, torch.zeros_like(prob), prob).view(-1).float()]


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        b, h, s, d, dim = (case[x] for x in ("b", "h", "s", "d", "dim"))
        return {"bytes": 8 * b * h * s * d + (4 * b * s if case["far"] else 0) + 4 * dim, "flops": 3 * b * h * s * dim}
    if kind == "append":
        total = sum(_sequences(case)[1])
        h, hkv, d, dim = (case[x] for x in ("h", "hkv", "d", "dim"))
        return {"bytes": 8 * total * d * (h + 2 * hkv) + 4 * dim + (4 * total if case["tree"] else 0),
                "flops": 3 * total * (h + hkv) * dim}
    if kind == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * (-(-k // 2)) + n * groups * (5 if case["zeros"] else 4) + 4 * m * (n + k) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    return {"bytes": 4 * case["rows"] * case["vocab"] + 12 * case["rows"], "flops": 3 * case["rows"] * case["vocab"]}


# ---- the same in 64 bits, from the definition ----------------------------------------------


def _exact_turn(x, positions, case, sign):
    """x [rows, heads, D] as complex numbers times scale * exp(i angle)."""
    dim = case["dim"]
    f = torch.from_numpy(_freq(case)).cuda()
    turn = torch.polar(torch.full_like(f, _turn_scale(case)).expand(positions.shape[0], -1).contiguous(),
                       sign * positions.double()[:, None] * f)[:, None]
    out = x.double().clone()
    if case["interleaved"]:
        z = torch.view_as_complex(out[..., :dim].reshape(*x.shape[:2], dim // 2, 2).contiguous()) * turn
        out[..., :dim] = torch.view_as_real(z).reshape(*x.shape[:2], dim)
    else:
        z = torch.complex(out[..., :dim // 2], out[..., dim // 2:dim]) * turn
        out[..., :dim] = torch.cat([z.real, z.imag], -1)
    return out


def _exact_token(x, temperature, k, p, min_p, u):
    """One row: what is left is found by walking down the sorted logits."""
    if not np.any(x > -np.inf):
        return -1, 0.0
    if temperature <= 0:
        return int(np.flatnonzero(x == x.max())[0]), 1.0
    ids = np.argsort(-x, kind="stable")
    ids = ids[x[ids] > -np.inf]
    if k > 0:
        ids = ids[:k]
    w = np.exp((x[ids] - x[ids[0]]) / temperature)
    if p < 1:
        n = int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1
        ids, w = ids[:n], w[:n]
    on = w >= min_p
    ids, w = ids[on], w[on]
    by = np.argsort(ids)
    ids, w = ids[by], w[by]
    at = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), len(ids) - 1)
    return int(ids[at]), float(w[at] / w.sum())


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        v = x["x"] if case["heads_last"] else x["x"].transpose(1, 2)
        b, s, h, d = v.shape
        pos = x["positions"] if "positions" in x else torch.arange(s, device="cuda").repeat(b, 1)
        out = _exact_turn(v.reshape(b * s, h, d), pos.reshape(-1), case, -1.0 if case["back"] else 1.0).view(b, s, h, d)
        return out if case["heads_last"] else out.transpose(1, 2).contiguous()
    if kind == "append":
        lens, news = _sequences(case)
        positions, slots, pages = [], [], []
        table = x["table"].cpu().numpy()
        for b, (length, n) in enumerate(zip(lens, news)):
            depth = list(range(n))
            if case["tree"]:
                parents = _parents(case)[b]
                for i, p in enumerate(parents):
                    depth[i] = 0 if p < 0 else depth[p] + 1
            positions += [length - n + t for t in depth]
            for j in range(length - n, length):
                pages.append(int(table[b, j // case["page"]]))
                slots.append(j % case["page"])
        pos, a, t = (torch.tensor(y, device="cuda") for y in (positions, pages, slots))
        k, v = x["k"].double(), x["v"].double()
        k[a, :, t] = _exact_turn(x["new_k"], pos, case, 1.0)
        v[a, :, t] = x["new_v"].double()
        return [_exact_turn(x["q"], pos, case, 1.0), k, v]
    if kind == "w4":
        n, k, group = case["n"], case["k"], case["group"]
        c = x["codes"].long()
        code = torch.empty(n, 2 * c.shape[1], dtype=torch.float64, device="cuda")
        code[:, 0::2], code[:, 1::2] = (c % 16).double(), (c // 16).double()
        y = torch.zeros(case["m"], n, dtype=torch.float64, device="cuda")
        for g in range(-(-k // group)):
            lo, hi = g * group, min(k, (g + 1) * group)
            zero = x["zero"][:, g].double() if "zero" in x else torch.full((n,), 8.0, dtype=torch.float64, device="cuda")
            w = (code[:, lo:hi] - zero[:, None]) * x["scale"][:, g].double()[:, None]
            y += x["x"][:, lo:hi].double() @ w.t().contiguous()
        if case["bias"]:
            y += x["bias"].double()
        if case["act"] == "relu":
            y.clamp_min_(0.0)
        if case["act"] == "gelu":
            y = y / (1.0 + torch.exp(-2.0 * 0.7978845608 * (y + 0.044715 * y ** 3)))
        return y
    logits, u = x["logits"].cpu().numpy().astype(np.float64), x["u"].cpu().numpy().astype(np.float64)
    tokens, probs = [], []
    for i, (t, k, p, min_p) in enumerate(_rules(case)):
        f = np.float32
        token, prob = _exact_token(logits[i], float(f(t)), k, float(f(p)), float(f(min_p)), u[i])
        tokens.append(token)
        probs.append(prob)
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)]
