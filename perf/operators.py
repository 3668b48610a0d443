"""Timed cases of the paged key/value cache and of the attention that reads it.

Each case is one pass through the operators as a serving program makes it:

  window   attention with a sliding window and sinks over a paged cache,     bch_sdpa_paged
           one new token a sequence, a chunk of a prompt, or a whole one
           (window 0: every key up to the row's own)
  dense    the same over dense [B, H, S, D] operands                         Tensor.sliding_window_attention
  tree     attention of a tree of drafted tokens over a paged cache          bch_sdpa_paged with parents
  append   new tokens' keys and values into the cache's pages                bch_kv_append
  fork     pages copied to others, as a forked sequence needs them           bch_kv_copy_pages
  keep     keys moved down in their sequences: the accepted drafts of a      bch_kv_append, bch_kv_keep
           step that appended all of them ("drafts"), or the sinks and the
           last keys of a long sequence ("evict")

Sequence b holds len[b] keys, its n new tokens among them, in pages that the
table names in order.  Row i of its n is at position len[b] - n + i, drafted
tokens at the position behind their parent's.  A key is visible to a row when
it is not behind it (for drafts: committed, or the row itself or one of its
ancestors) and lies less than `window` positions back or in the first `sinks`.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # one short conversation, one token: launch latency counts
        {"name": "window_decode_one", "kind": "window", "b": 1, "h": 8, "hkv": 8, "d": 64, "len": 300, "new": 1,
         "page": 16, "window": 256, "sinks": 4, "ragged": False},
        # a decode step of 32 conversations of very different lengths, 8 key/value heads for 32 query heads
        {"name": "window_decode_batch", "kind": "window", "b": 32, "h": 32, "hkv": 8, "d": 128, "len": 16384, "new": 1,
         "page": 64, "window": 4096, "sinks": 4, "ragged": True},
        # a decode step over long documents, every key read
        {"name": "decode_long", "kind": "window", "b": 4, "h": 32, "hkv": 8, "d": 128, "len": 65536, "new": 1,
         "page": 64, "window": 0, "sinks": 0, "ragged": False},
        # a whole prompt through the window: the largest case
        {"name": "window_prefill", "kind": "window", "b": 1, "h": 32, "hkv": 8, "d": 128, "len": 16384, "new": 16384,
         "page": 64, "window": 4096, "sinks": 4, "ragged": False},
        # chunks of prompts of odd lengths behind what their sequences hold already, a narrow odd head
        {"name": "window_chunks", "kind": "window", "b": 7, "h": 12, "hkv": 4, "d": 80, "len": 4099, "new": 517,
         "page": 16, "window": 512, "sinks": 1, "ragged": True},
        # dense operands with as many key/value heads as query heads, bench.py's attention shape
        {"name": "window_dense", "kind": "dense", "b": 4, "h": 32, "hkv": 32, "d": 128, "sq": 2048, "skv": 2048,
         "window": 512, "sinks": 4},
        # eight drafted tokens of one conversation: launch latency counts
        {"name": "tree_one", "kind": "tree", "b": 1, "h": 8, "hkv": 8, "d": 64, "len": 500, "new": 8, "page": 16,
         "window": 0, "sinks": 0, "ragged": False},
        # a verification step of 16 conversations with 64 drafts each
        {"name": "tree_batch", "kind": "tree", "b": 16, "h": 32, "hkv": 8, "d": 128, "len": 8192, "new": 64, "page": 64,
         "window": 0, "sinks": 0, "ragged": True},
        # the decode step's tokens into their pages
        {"name": "append_decode", "kind": "append", "b": 32, "hkv": 8, "d": 128, "len": 1024, "new": 1, "page": 16,
         "ragged": True},
        # prompts into their pages
        {"name": "append_prefill", "kind": "append", "b": 8, "hkv": 8, "d": 128, "len": 4096, "new": 4096, "page": 64,
         "ragged": True},
        # pages of forked sequences copied
        {"name": "fork_pages", "kind": "fork", "layers": 1, "hkv": 8, "d": 128, "page": 16, "pages": 1500},
        # drafts of every layer appended, the accepted ones kept
        {"name": "keep_drafts", "kind": "keep", "mode": "drafts", "layers": 4, "b": 16, "hkv": 8, "d": 128, "len": 700,
         "new": 64, "page": 16, "ragged": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of them."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 9e11 and w["bytes"] <= 2e9 and _plain_pairs(case) <= 8e9:
            return case


def _draw(rng):
    kind = rng.choice(["window", "window", "window", "dense", "tree", "tree", "append", "fork", "keep"])
    hkv = rng.choice([1, 2, 4, 8])
    h = hkv * rng.choice([1, 1, 2, 4, 4, 8])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 128])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 64, 128, 256])
    ragged = rng.random() < 0.7
    window = 0 if rng.random() < 0.25 else _log(rng, 16, 8192)
    sinks = 0 if window == 0 else rng.choice([0, 1, 4, 4, 33])
    if kind == "window":
        length = _log(rng, 1, 32768)
        new = 1 if rng.random() < 0.5 else _log(rng, 1, length)
        return {"kind": kind, "b": _log(rng, 1, 48 if new <= 64 else 8), "h": h, "hkv": hkv, "d": d, "len": length,
                "new": new, "page": page, "window": window, "sinks": sinks, "ragged": ragged}
    if kind == "dense":
        skv = _log(rng, 16, 8192)
        return {"kind": kind, "b": rng.randint(1, 4), "h": h, "hkv": hkv, "d": d,
                "sq": skv if rng.random() < 0.7 else _log(rng, 1, skv), "skv": skv, "window": window, "sinks": sinks}
    if kind == "tree":
        new = _log(rng, 2, 128)
        return {"kind": kind, "b": _log(rng, 1, 32), "h": h, "hkv": hkv, "d": d, "len": _log(rng, new, 16384), "new": new,
                "page": page, "window": window, "sinks": sinks, "ragged": ragged}
    if kind == "append":
        length = _log(rng, 1, 8192)
        return {"kind": kind, "b": _log(rng, 1, 32), "hkv": hkv, "d": d, "len": length,
                "new": 1 if rng.random() < 0.4 else _log(rng, 1, length), "page": page, "ragged": ragged}
    if kind == "fork":
        return {"kind": kind, "layers": rng.choice([1, 1, 4]), "hkv": hkv, "d": d, "page": page,
                "pages": _log(rng, 1, 1500)}
    if rng.random() < 0.5:
        new = _log(rng, 2, 128)
        return {"kind": kind, "mode": "drafts", "layers": rng.choice([1, 4, 8]), "b": _log(rng, 1, 16), "hkv": hkv, "d": d,
                "len": _log(rng, new, 2048), "new": new, "page": page, "ragged": ragged}
    keep = _log(rng, 8, 1024)
    return {"kind": kind, "mode": "evict", "layers": rng.choice([1, 4]), "b": _log(rng, 1, 8), "hkv": hkv, "d": d,
            "len": 2 * keep + 8 + _log(rng, 1, 1024), "new": keep, "page": page, "ragged": False}


# ---- what a case's sequences are ------------------------------------------------------


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _sequences(case):
    """Keys and new tokens of every sequence: the first one's are the case's, ragged ones' are anything up to it."""
    r = _rng(case)
    lens, news = [case["len"]], [min(case["new"], case["len"])]
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
    out = []
    for n in _sequences(case)[1]:
        # a few branches at the root, then mostly deeper
        out.append([-1 if i == 0 or r.random() < 0.1 else r.randint(max(0, i - 8), i - 1) for i in range(n)])
    return out


def _kept(case):
    """For each sequence the positions kept, and the position that the first of them goes to."""
    r = _rng(case)
    lens, news = _sequences(case)
    if case["mode"] == "evict":  # the sinks and the last keys; those do not reach into what is written
        return [list(range(length - new, length)) for length, new in zip(lens, news)], [4] * len(lens)
    keep, to = [], []
    for parents, length, n in zip(_parents(case), lens, news):
        path, x = [], r.randint(0, n - 1) if n else -1
        while x >= 0:
            path.append(length - n + x)
            x = parents[x]
        keep.append(path[::-1])
        to.append(length - n)
    return keep, to


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _plain_pairs(case):
    """Scores that a form without skipping computes."""
    if case["kind"] == "dense":
        return case["b"] * case["h"] * case["sq"] * case["skv"]
    if case["kind"] not in ("window", "tree"):
        return 0
    return case["h"] * sum(length * n for length, n in zip(*_sequences(case)))


# ---- inputs ---------------------------------------------------------------------------


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda").reshape(-1)


def _inputs(case, seed):
    """The case's inputs as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind, d, hkv = case["kind"], case["d"], case["hkv"]
    if kind == "dense":
        b, h, sq, skv = case["b"], case["h"], case["sq"], case["skv"]
        return {"q": normal(b, h, sq, d), "k": normal(b, hkv, skv, d), "v": normal(b, hkv, skv, d)}
    page, layers = case["page"], case.get("layers", 1)
    x = {}
    if kind == "fork":
        n = case["pages"]
        pages = 2 * n
        order = torch.randperm(pages, generator=g, device="cuda").cpu().numpy().astype(np.int32)
        x["src"], x["dst"] = order[:n].copy(), order[n:].copy()
    else:
        lens, news = _sequences(case)
        held = [-(-length // page) for length in lens]
        pages = sum(held) + max(1, sum(held) // 16)
        width = max(1, max(held))
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(held):
            table[b, :n] = order[at:at + n]
            at += n
        start = np.concatenate([[0], np.cumsum(news)]).tolist()
        x.update(table=table, len=_i32(lens), start=_i32(start))
        total = start[-1]
        if kind in ("window", "tree"):
            x["q"] = normal(total, case["h"], d)
        if kind == "tree":
            x["parent"] = _i32([p for seq in _parents(case) for p in seq])
        if kind == "append" or case.get("mode") == "drafts":
            x["new_k"], x["new_v"] = normal(layers, total, hkv, d), normal(layers, total, hkv, d)
        if kind == "keep":
            keep, to = _kept(case)
            x["keep"] = _i32([p for seq in keep for p in seq])
            x["keep_start"] = _i32(np.concatenate([[0], np.cumsum([len(s) for s in keep])]).tolist())
            x["to"] = _i32(to)
    # pools as the cache lays them out: a head's keys of a page side by side
    x["k"], x["v"] = normal(layers, pages, hkv, page, d), normal(layers, pages, hkv, page, d)
    return x


class _Span:
    """Device memory that another object owns, for torch.as_tensor."""

    def __init__(self, ptr, shape, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (ptr, False), "version": 2}


def _view(t):
    """A Tensor's buffer as a torch tensor, without a copy."""
    return torch.as_tensor(_Span(t.ptr, t.shape(), t), device="cuda")


def _p(x):
    return ctypes.c_void_p(x.data_ptr())


def _handles(case, x):
    """What a serving program keeps beside its buffers: the cache's description and the step's batch."""
    from barracuda_amd import Tensor, _native, get_device
    dev = get_device()
    own_state = {"dev": dev, "lib": _native.load()}
    if case["kind"] == "dense":
        for name in ("q", "k", "v"):
            t = Tensor.empty(list(x[name].shape), dev)
            _view(t).copy_(x[name])
            own_state["t" + name] = t
        return own_state
    layers, pages, hkv, page, d = x["k"].shape
    layout = _native.AttnLayout(hkv * page * d, page * d, d)
    own_state["kv"] = [
        _native.KvPages(x["k"][i].data_ptr(), x["v"][i].data_ptr(), layout, layout, pages, page, hkv, d,
                        x["table"].data_ptr() if "table" in x else None, x["table"].shape[1] if "table" in x else 0)
        for i in range(layers)]
    if "len" in x:
        lens, news = _sequences(case)
        own_state["batch"] = _native.KvBatch(len(lens), sum(news), max(news), max(lens), x["start"].data_ptr(),
                                             x["len"].data_ptr())
    if "q" in x:
        own_state["rows"] = _native.AttnLayout(0, d, case["h"] * d)
        own_state["o"] = torch.empty_like(x["q"])
    if "new_k" in x:
        own_state["new"] = _native.AttnLayout(0, d, hkv * d)
    return own_state


def prepare(case, seed):
    """Inputs, cache, tables and handles in HBM; the output that a serving loop holds."""
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
    if kind == "dense":
        return _view(s["tq"].sliding_window_attention(s["tk"], s["tv"], case["window"], case["sinks"]))
    kv = s["kv"]
    if kind in ("window", "tree"):
        parent = _p(x["parent"]) if kind == "tree" else None
        dev.check(lib.bch_sdpa_paged(dev.ctx, kv[0], s["batch"], case["h"], 1.0 / math.sqrt(case["d"]), case["window"],
                                     case["sinks"], parent, _p(x["q"]), s["rows"], _p(s["o"]), s["rows"]), "attention")
        return s["o"]
    stride = x["k"].stride(0)
    if "new_k" in x:
        for i in range(len(kv)):
            dev.check(lib.bch_kv_append(dev.ctx, kv[i], s["batch"], _p(x["new_k"][i]), s["new"], _p(x["new_v"][i]),
                                        s["new"]), "append")
    if kind == "fork":
        src, dst = (x[p].ctypes.data_as(ctypes.POINTER(ctypes.c_int)) for p in ("src", "dst"))
        dev.check(lib.bch_kv_copy_pages(dev.ctx, kv[0], len(kv), stride, stride, len(x["src"]), src, dst), "copy_pages")
    elif kind == "keep":
        dev.check(lib.bch_kv_keep(dev.ctx, kv[0], len(kv), stride, stride, len(x["to"]), len(x["keep"]),
                                  _p(x["keep_start"]), _p(x["keep"]), _p(x["to"])), "keep")
    return [x["k"], x["v"]]


# the plain form: gathers, products, exponentials and sums in float32


def _gather(pool, table, length):
    """A sequence's keys or values, [Hkv, length, D]."""
    hkv, page, d = pool.shape[1:]
    n = -(-length // page)
    return pool[table[:n].long()].transpose(0, 1).reshape(hkv, n * page, d)[:, :length].contiguous()


def _attend(q, k, v, visible, scale):
    """q [Hkv, G, n, D], k and v [Hkv, L, D], visible(rows) -> [rows, L] of truth values."""
    hkv, g, n, d = q.shape
    out = torch.empty_like(q)
    kt = k.transpose(1, 2).contiguous()
    step = max(1, (1 << 28) // (hkv * g * k.shape[1]))
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        mask = ~visible(torch.arange(r0, r1, device=q.device))
        s = torch.matmul(q[:, :, r0:r1].reshape(hkv, g * (r1 - r0), d), kt).view(hkv, g, r1 - r0, -1) * scale
        s.masked_fill_(mask, -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        p = s.sub_(m).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hkv, g * (r1 - r0), -1), v).view(hkv, g, r1 - r0, d)
        out[:, :, r0:r1] = torch.where(total > 0, o / torch.where(total > 0, total, torch.ones_like(total)),
                                       torch.zeros_like(o))
    return out


def _chain(first, length, window, sinks):
    """Which keys row i at position first + i sees."""
    key = torch.arange(length, device="cuda")

    def visible(rows):
        pos = (first + rows)[:, None]
        see = key[None, :] <= pos
        if window:
            see &= (pos - key[None, :] < window) | (key[None, :] < sinks)
        return see
    return visible


def _tree(parent, first, length, window, sinks):
    """The same for drafts: their ancestors by repeated squaring of the parent relation."""
    n = parent.shape[0]
    row = torch.arange(n, device="cuda")
    reach = torch.eye(n, device="cuda")
    reach += (parent.long()[:, None] == row[None, :]).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    pos = first + (reach.sum(1).long() - 1)
    key_pos = torch.arange(length, device="cuda")
    key_pos[first:] = pos

    def visible(rows):
        see = torch.ones(rows.shape[0], length, dtype=torch.bool, device="cuda")
        see[:, first:] = reach[rows] > 0
        if window:
            see &= (pos[rows][:, None] - key_pos[None, :] < window) | (key_pos[None, :] < sinks)
        return see
    return visible


def _slots(x, page, which, positions):
    """Page and slot of each position of the sequences `which`."""
    return x["table"][which, positions // page].long(), positions % page


def _run_plain(case, x):
    kind = case["kind"]
    if kind == "dense":
        q, k, v = x["q"], x["k"], x["v"]
        b, h, sq, d = q.shape
        hkv, skv = k.shape[1:3]
        see = _chain(skv - sq, skv, case["window"], case["sinks"])
        return torch.stack([_attend(q[i].reshape(hkv, h // hkv, sq, d), k[i], v[i], see, 1.0 / math.sqrt(d))
                            .reshape(h, sq, d) for i in range(b)])
    layers, page, hkv, d = x["k"].shape[0], case["page"], case["hkv"], case["d"]
    if kind in ("window", "tree"):
        lens, news = _sequences(case)
        out = torch.empty_like(x["q"])
        at = 0
        for b, (length, n) in enumerate(zip(lens, news)):
            if n:
                k, v = (_gather(x[p][0], x["table"][b], length) for p in ("k", "v"))
                q = x["q"][at:at + n].view(n, hkv, -1, d).permute(1, 2, 0, 3)
                if kind == "tree":
                    see = _tree(x["parent"][at:at + n], length - n, length, case["window"], case["sinks"])
                else:
                    see = _chain(length - n, length, case["window"], case["sinks"])
                out[at:at + n] = _attend(q, k, v, see, 1.0 / math.sqrt(d)).permute(2, 0, 1, 3).reshape(n, -1, d)
            at += n
        return out
    if "new_k" in x:
        start = x["start"].long()
        n = start[1:] - start[:-1]
        which = torch.repeat_interleave(torch.arange(n.shape[0], device="cuda"), n, output_size=x["new_k"].shape[1])
        positions = (x["len"].long() - n - start[:-1])[which] + torch.arange(which.shape[0], device="cuda")
        at, slot = _slots(x, page, which, positions)
        for i in range(layers):
            x["k"][i][at, :, slot] = x["new_k"][i]
            x["v"][i][at, :, slot] = x["new_v"][i]
    if kind == "fork":
        src, dst = (torch.as_tensor(x[p]).long().cuda() for p in ("src", "dst"))
        for i in range(layers):
            x["k"][i][dst] = x["k"][i][src]
            x["v"][i][dst] = x["v"][i][src]
    elif kind == "keep":
        start = x["keep_start"].long()
        n = start[1:] - start[:-1]
        which = torch.repeat_interleave(torch.arange(n.shape[0], device="cuda"), n, output_size=x["keep"].shape[0])
        to = (x["to"].long() - start[:-1])[which] + torch.arange(which.shape[0], device="cuda")
        at, slot = _slots(x, page, which, x["keep"].long())
        at2, slot2 = _slots(x, page, which, to)
        for i in range(layers):
            x["k"][i][at2, :, slot2] = x["k"][i][at, :, slot]
            x["v"][i][at2, :, slot2] = x["v"][i][at, :, slot]
    return [x["k"], x["v"]]


# ---- what a pass cannot do without --------------------------------------------------------


def _seen(pos, window, sinks):
    """Keys that a row at position pos sees of an unbranched sequence."""
    if not window or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def _read(first, length, window, sinks):
    """Keys of a sequence that any of its rows from position first on sees."""
    lo = max(0, first - window + 1) if window else 0
    return length - lo + min(sinks, lo)


def work(case):
    kind, d, hkv = case["kind"], case["d"], case["hkv"]
    if kind == "fork":
        return {"bytes": 16 * case["layers"] * case["pages"] * case["page"] * hkv * d, "flops": 0}
    if kind == "dense":
        b, h, sq, skv, w, s = (case[x] for x in ("b", "h", "sq", "skv", "window", "sinks"))
        pairs = sum(_seen(p, w, s) for p in range(skv - sq, skv))
        return {"bytes": 8 * b * d * (h * sq + hkv * _read(skv - sq, skv, w, s)), "flops": 4 * b * h * d * pairs}
    lens, news = _sequences(case)
    if kind == "append":
        return {"bytes": 16 * hkv * d * sum(news), "flops": 0}
    if kind == "keep":
        moved = sum(len(s) for s in _kept(case)[0])
        new = sum(news) if case["mode"] == "drafts" else 0
        return {"bytes": 16 * case["layers"] * hkv * d * (moved + new), "flops": 0}
    h, w, s = case["h"], case["window"], case["sinks"]
    pairs = read = 0
    for b, (length, n) in enumerate(zip(lens, news)):
        if n == 0:
            continue
        first = length - n
        if kind == "tree":
            pairs += sum(_seen(first + x, w, s) for x in _depths(_parents(case)[b]))
        else:
            pairs += sum(_seen(p, w, s) for p in range(first, length))
        read += _read(first, length, w, s)
    return {"bytes": 8 * d * (h * sum(news) + hkv * read), "flops": 4 * h * d * pairs}


# ---- the same in 64 bits, from the definition ----------------------------------------------


def _ancestors(parents):
    """Of each draft the list of itself and its ancestors."""
    out = []
    for i, p in enumerate(parents):
        out.append([i] + (out[p] if p >= 0 else []))
    return out


def _exact_rows(q, k, v, see, d):
    """softmax(q k^T / sqrt(d)) v over the keys that see [rows, keys] allows, for one head."""
    s = (q @ k.T.contiguous()) / math.sqrt(d)
    e = torch.where(see, torch.exp(s - torch.where(see, s, torch.full_like(s, -1e300)).max(1, keepdim=True)[0]),
                    torch.zeros_like(s))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, (e @ v) / total.clamp_min(1e-300), torch.zeros_like(q))


def _exact_sequence(q, k, v, case, parents):
    """q [n, H, D], k and v [length, Hkv, D], all float64; a few hundred rows and the keys near them at a time."""
    n, h, d = q.shape
    length, hkv = k.shape[:2]
    w, sinks = case["window"], case["sinks"]
    first = length - n
    out = torch.zeros_like(q)
    for r0 in range(0, n, 512):
        r1 = min(n, r0 + 512)
        if parents is None:
            pos = list(range(first + r0, first + r1))
            lo, hi = (max(0, pos[0] - w + 1) if w else 0), pos[-1] + 1
        else:
            depth = _depths(parents)
            pos = [first + depth[i] for i in range(r0, r1)]
            lo, hi = (max(0, first - w + 1) if w else 0), length
        keys = sorted(set(range(min(sinks, hi))) | set(range(lo, hi)))
        where = {j: x for x, j in enumerate(keys)}
        kp = np.array(keys)
        see = np.zeros((r1 - r0, len(keys)), dtype=bool)
        if parents is None:
            for x, p in enumerate(pos):
                see[x] = kp <= p
                if w:
                    see[x] &= (kp > p - w) | (kp < sinks)
        else:
            chains = _ancestors(parents)
            for x, p in enumerate(pos):
                see[x] = kp < first
                if w:
                    see[x] &= (kp > p - w) | (kp < sinks)
                for a in chains[r0 + x]:
                    at = first + depth[a]
                    if not w or p - at < w or at < sinks:
                        see[x, where[first + a]] = True
        see = torch.from_numpy(see).cuda()
        index = torch.from_numpy(kp).cuda()
        for head in range(h):
            kv = head // (h // hkv)
            out[r0:r1, head] = _exact_rows(q[r0:r1, head].contiguous(), k[index, kv].contiguous(),
                                           v[index, kv].contiguous(), see, d)
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "dense":
        q, k, v = (x[p].double().transpose(1, 2) for p in ("q", "k", "v"))
        return torch.stack([_exact_sequence(q[i], k[i], v[i], case, None).transpose(0, 1) for i in range(case["b"])])
    page = case["page"]
    if kind == "fork":
        k, v = x["k"].double(), x["v"].double()
        for pool in (k, v):
            old = pool.clone()
            for a, b in zip(x["src"].tolist(), x["dst"].tolist()):
                pool[:, b] = old[:, a]
        return [k, v]
    lens, news = _sequences(case)
    table = x["table"].cpu().numpy()

    def rows(pool, b, positions):
        """The pool's rows of these positions, one index a page and one a slot."""
        p = np.asarray(positions, dtype=np.int64)
        return torch.from_numpy(table[b, p // page].astype(np.int64)).cuda(), torch.from_numpy(p % page).cuda()

    if kind in ("window", "tree"):
        parents = _parents(case) if kind == "tree" else [None] * len(lens)
        out, at = [], 0
        for b, (length, n) in enumerate(zip(lens, news)):
            if n:
                a, s = rows(x["k"], b, range(length))
                out.append(_exact_sequence(x["q"][at:at + n].double(), x["k"][0][a, :, s].double(),
                                           x["v"][0][a, :, s].double(), case, parents[b]))
            at += n
        return torch.cat(out)
    k, v = x["k"].double(), x["v"].double()
    if "new_k" in x:
        at = 0
        for b, (length, n) in enumerate(zip(lens, news)):
            a, s = rows(k, b, range(length - n, length))
            for layer in range(k.shape[0]):
                k[layer][a, :, s] = x["new_k"][layer, at:at + n].double()
                v[layer][a, :, s] = x["new_v"][layer, at:at + n].double()
            at += n
    if kind == "keep":
        keep, to = _kept(case)
        for b in range(len(lens)):
            if not keep[b]:
                continue
            a, s = rows(k, b, keep[b])
            a2, s2 = rows(k, b, range(to[b], to[b] + len(keep[b])))
            for layer in range(k.shape[0]):
                for pool in (k, v):
                    pool[layer][a2, :, s2] = pool[layer][a, :, s].clone()
    return [k, v]
