"""KvCache: a paged key/value cache that several sequences share.

The reference keeps no cache (its attention ops take whole dense K and V,
ops/causal_attn/mod.rs:64-158, ops/grouped_query_attention/mod.rs:52-147);
this stands beside them for programs that serve sequences token by token.

The pools K and V are [layers, pages, kv_heads, page_size, head_dim] in HBM.
A sequence is a list of pages, the same in every layer; its key j is slot
j % page_size of its page j // page_size.  Pages are counted: a fork shares its
parent's, and a page that more than one sequence holds is copied before one of
them writes into it.  The bookkeeping is on the host; what a step's kernels
need of it (page table, starts, lengths, the drafts' parents) is uploaded once
per step and serves every layer.  A cache is for one thread at a time.

    cache = KvCache(layers, pages, page_size, kv_heads, head_dim)
    a = cache.new_sequence()
    step = cache.batch([(a, 512)])                 # room for 512 new tokens
    for layer in range(layers):
        cache.append(step, layer, k, v)            # [total, kv_heads, head_dim]
        o = cache.attention(step, layer, q, window=4096, sinks=4)
    b = cache.fork(a)
    step = cache.batch([(a, 5), (b, 1)], parents=[[-1, 0, 0, 1, 1], [-1]])
    ...                                            # append and attention as above
    cache.keep(step, [[0, 2], [0]])                # the accepted drafts stay
    cache.evict(a, window=4096, sinks=4)           # pages no later token sees
    cache.free(b)
    cache.compact()                                # live pages to the front
"""
from __future__ import annotations

import ctypes as C
from typing import Iterable, Sequence

import numpy as np

from . import _native as N
from .error import DeviceError, InvalidInput, InvalidOperation, OutOfMemory, ShapeMismatch
from .tensor import HipDevice, Tensor, _Buffer, _I32_MAX, get_device

__all__ = ["KvCache", "KvStep"]

MAX_DRAFTS = 128  # of one sequence's tree
_MAX_KEYS = 2**31 - 256  # of a sequence
_KEEP_SEQUENCES, _KEEP_LAYERS = 65535, 32767  # of one bch_kv_keep


class _I32:
    """int32 arrays side by side in one device buffer, uploaded together."""

    def __init__(self, device: HipDevice, *arrays):
        arrays = [np.ascontiguousarray(a, dtype=np.int32).reshape(-1) for a in arrays]
        self._buf = _Buffer(device, 4 * max(1, sum(a.size for a in arrays)))
        flat = np.concatenate(arrays)
        if flat.size:
            device.upload(self._buf.ptr, flat)
        self.ptrs, at = [], self._buf.ptr
        for a in arrays:
            self.ptrs.append(at)
            at += 4 * a.size


class KvStep:
    """The new tokens of one step: which sequences, and how many each.  Made by
    KvCache.batch; row start[i] .. start[i + 1] - 1 of the step's q, k, v and
    output are sequence i's.  A step serves until a page that an older step
    may name changes hands (keep, retain, truncate, evict, free, compact, or a
    batch that has to copy a shared page); its calls then raise
    InvalidOperation."""

    def __init__(self, cache: "KvCache", sequences: Sequence[int], counts: Sequence[int], parents):
        self._cache = cache
        self.sequences, self.counts = list(sequences), list(counts)
        lens = self._lens = [cache._seqs[s].length for s in sequences]
        self.start = np.concatenate([[0], np.cumsum(counts, dtype=np.int64)]).astype(np.int64)
        self.total = int(self.start[-1])
        width = max([1] + [len(cache._seqs[s].pages) for s in sequences])
        table = np.full((len(lens), width), -1, dtype=np.int32)
        for i, s in enumerate(sequences):
            table[i, :len(cache._seqs[s].pages)] = cache._seqs[s].pages
        flat = [] if parents is None else [p for tree in parents for p in tree]
        self._dev = _I32(cache.device, self.start, lens, table, flat)
        start, length, tab, par = self._dev.ptrs
        self._batch = N.KvBatch(len(lens), self.total, max([0] + self.counts), max([0] + lens), start, length)
        self._table, self._width = tab, width
        self._parents = C.c_void_p(par) if parents is not None else None
        # of each sequence with new tokens the evicted keys: the first, the end, and the keys before the new tokens
        self._gone = []
        for s, n, length in zip(sequences, counts, lens):
            if n and cache._seqs[s].evicted:
                at = [i for i, p in enumerate(cache._seqs[s].pages) if p < 0]
                if at:
                    self._gone.append((at[0] * cache.page_size, (at[-1] + 1) * cache.page_size, length - n))
        self._generation = cache._generation


class _Sequence:
    __slots__ = ("pages", "length", "evicted")

    def __init__(self):
        self.pages: list[int] = []  # -1: given back by evict
        self.length = 0
        self.evicted = False  # whether there may be such pages


class KvCache:
    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 device: HipDevice | None = None):
        dims = {"layers": layers, "num_pages": num_pages, "page_size": page_size, "kv_heads": kv_heads,
                "head_dim": head_dim}
        for name, v in dims.items():
            if not 1 <= v <= _I32_MAX:
                raise InvalidInput(f"KvCache: {name} must be at least 1 and fit 32 bits, got {v}")
        self.device = device or get_device()
        self.layers, self.num_pages, self.page_size = layers, num_pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        shape = [layers, num_pages, kv_heads, page_size, head_dim]
        self.k, self.v = Tensor.empty(shape, self.device), Tensor.empty(shape, self.device)
        page = kv_heads * page_size * head_dim
        self._layout = N.AttnLayout(page, page_size * head_dim, head_dim)
        self._layer = num_pages * page
        self._free = list(range(num_pages - 1, -1, -1))  # the lowest page last
        self._refs = [0] * num_pages
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0
        self._generation = 0

    # -- sequences ------------------------------------------------------------
    def new_sequence(self) -> int:
        """An empty sequence; its number is good for this cache until free."""
        self._seqs[self._next] = _Sequence()
        self._next += 1
        return self._next - 1

    def fork(self, sequence: int) -> int:
        """A sequence with the same keys, its pages shared until one of the two
        writes into them."""
        s, f = self._seq(sequence), self.new_sequence()
        self._seqs[f].pages, self._seqs[f].length, self._seqs[f].evicted = list(s.pages), s.length, s.evicted
        for p in s.pages:
            if p >= 0:
                self._refs[p] += 1
        return f

    def free(self, sequence: int) -> None:
        """Give a sequence's pages back."""
        s = self._seq(sequence)
        self._generation += 1
        for p in s.pages:
            self._drop(p)
        del self._seqs[sequence]

    def length(self, sequence: int) -> int:
        return self._seq(sequence).length

    def pages(self, sequence: int) -> list[int]:
        """The sequence's pages in order, -1 where evict gave one back."""
        return list(self._seq(sequence).pages)

    def free_pages(self) -> int:
        return len(self._free)

    # -- a step -----------------------------------------------------------------
    def batch(self, items: Iterable[tuple[int, int]], parents: Sequence[Sequence[int]] | None = None) -> KvStep:
        """Make room for `count` new tokens of each (sequence, count): pages are
        taken from the free ones, and a shared page that the first of them
        falls into is copied.  OutOfMemory, with nothing changed, if there are
        too few.  With `parents` the new tokens of a sequence are a tree of at
        most 128 drafts: parents[i][j] is the draft that draft j follows, -1 the
        last committed token."""
        items = [(int(s), int(n)) for s, n in items]
        seqs = [self._seq(s) for s, _ in items]
        if len({s for s, _ in items}) != len(items):
            raise InvalidInput("KvCache.batch: a sequence is named twice")
        for s, n in items:
            if n < 0 or self._seqs[s].length + n > _MAX_KEYS:
                raise InvalidInput(f"KvCache.batch: {n} new tokens for sequence {s}")
        if sum(n for _, n in items) > _I32_MAX:
            raise InvalidInput("KvCache.batch: too many new tokens")
        if parents is not None:
            self._check_parents(items, parents)
        ps = self.page_size
        need, tails = 0, []
        for (_, n), s in zip(items, seqs):
            need += -(-(s.length + n) // ps) - -(-s.length // ps)
            if n and s.length % ps:
                if s.pages[-1] < 0:
                    raise InvalidOperation("KvCache.batch", "the page that the new tokens fall into has been evicted")
                tails.append((s, len(s.pages) - 1))
        self._own_pages(tails, need)
        old = [s.length for s in seqs]
        for (_, n), s in zip(items, seqs):
            s.length += n
            while len(s.pages) * ps < s.length:
                s.pages.append(self._take())
        try:
            return KvStep(self, [s for s, _ in items], [n for _, n in items], parents)
        except BaseException:
            for s, length in zip(seqs, old):
                self._cut(s, length)
            raise

    def append(self, step: KvStep, layer: int, k: Tensor, v: Tensor) -> None:
        """The step's keys and values, [total, kv_heads, head_dim], into their pages."""
        self._check_step("KvCache.append", step, layer)
        shape = [step.total, self.kv_heads, self.head_dim]
        for t in (k, v):
            if t.shape() != shape:
                raise ShapeMismatch(shape, t.shape())
        self._own(k, v)
        if step.total == 0:
            return
        row = N.AttnLayout(0, self.head_dim, self.kv_heads * self.head_dim)
        dev = self.device
        with dev._lock:
            dev.check(dev._lib.bch_kv_append(dev.ctx, self._pages(step, layer), step._batch, C.c_void_p(k.ptr), row,
                                             C.c_void_p(v.ptr), row), "kv_append")

    def attention(self, step: KvStep, layer: int, q: Tensor, window: int = 0, sinks: int = 0,
                  scale: float | None = None) -> Tensor:
        """softmax(scale q K^T) V of the step's rows, q [total, heads, head_dim]
        with heads a multiple of kv_heads, scale 1/sqrt(head_dim) unless given.
        A row sees the keys up to its own (a draft: the committed ones, its
        ancestors and itself); with window > 0 only those less than `window`
        positions back and the first `sinks`.  InvalidOperation if one of them
        has been evicted."""
        self._check_step("KvCache.attention", step, layer)
        shape = q.shape()
        if len(shape) != 3 or shape[0] != step.total or shape[2] != self.head_dim:
            raise ShapeMismatch([step.total, self.kv_heads, self.head_dim], shape)
        heads = shape[1]
        if heads == 0 or heads % self.kv_heads != 0:
            raise InvalidInput(f"num_q_heads ({heads}) must be divisible by num_kv_heads ({self.kv_heads})")
        if window < 0 or sinks < 0:
            raise InvalidInput(f"window ({window}) and sinks ({sinks}) must not be negative")
        for begin, end, committed in step._gone:
            if window == 0 or begin < sinks or end > committed - window + 1:
                raise InvalidOperation("KvCache.attention", f"a row would see keys that have been evicted (of {begin} to "
                                       f"{end - 1}, {committed} keys before its own, window {window}, sinks {sinks})")
        self._own(q)
        out = Tensor.empty(shape, self.device)
        if step.total == 0:
            return out
        if scale is None:
            scale = float(np.float32(1.0) / np.sqrt(np.float32(self.head_dim)))
        row = N.AttnLayout(0, self.head_dim, heads * self.head_dim)
        dev = self.device
        with dev._lock:
            dev.check(dev._lib.bch_sdpa_paged(dev.ctx, self._pages(step, layer), step._batch, heads, scale,
                                              min(int(window), _I32_MAX), min(int(sinks), _I32_MAX), step._parents,
                                              C.c_void_p(q.ptr), row, C.c_void_p(out.ptr), row), "paged attention")
        return out

    # -- giving keys up ------------------------------------------------------------
    def keep(self, step: KvStep, kept: Sequence[Sequence[int]]) -> None:
        """Of each sequence's new tokens of `step` keep the ones listed
        (ascending, counted from the sequence's first): their keys move down
        behind the committed ones, the others and their pages are given up."""
        self._check_step("KvCache.keep", step, 0)
        if len(kept) != len(step.sequences):
            raise InvalidInput(f"KvCache.keep: {len(kept)} lists for {len(step.sequences)} sequences")
        if any(self._seqs[s].length != length for s, length in zip(step.sequences, step._lens)):
            raise InvalidOperation("KvCache.keep", "a later step has added tokens behind this one's")
        moves = []
        for s, n, ids in zip(step.sequences, step.counts, kept):
            ids = [int(x) for x in ids]
            if any(not 0 <= x < n for x in ids) or any(a >= b for a, b in zip(ids, ids[1:])):
                raise InvalidInput(f"KvCache.keep: {ids} does not ascend within {n} new tokens")
            first = self._seqs[s].length - n
            moves.append((s, first, [first + x for x in ids]))
        self._move(moves)

    def retain(self, sequence: int, positions: Sequence[int]) -> None:
        """Keep only the keys at these positions (ascending); they close up to
        positions 0, 1, ... and the pages behind them are given up."""
        s, positions = self._seq(sequence), [int(x) for x in positions]
        if any(not 0 <= x < s.length for x in positions) or any(a >= b for a, b in zip(positions, positions[1:])):
            raise InvalidInput(f"KvCache.retain: positions must ascend within {s.length} keys")
        if any(s.pages[x // self.page_size] < 0 for x in positions):
            raise InvalidOperation("KvCache.retain", "a key to keep is in a page that has been evicted")
        same = next((i for i, x in enumerate(positions) if x != i), len(positions))
        self._move([(sequence, same, positions[same:])])

    def truncate(self, sequence: int, length: int) -> None:
        """Give up all but the first `length` keys.  Windows then reach further
        back than before: into evicted pages, where attention is refused."""
        s = self._seq(sequence)
        if not 0 <= length <= s.length:
            raise InvalidInput(f"KvCache.truncate: length {length} of a sequence of {s.length}")
        self._generation += 1
        self._cut(s, length)

    def evict(self, sequence: int, window: int, sinks: int = 0) -> int:
        """Give back the pages whose keys no later token sees through this
        window and these sinks; the other keys keep their positions.  Returns
        the number of pages given back.  Attention of a later token that would
        see one of their keys all the same (through a larger window, with more
        sinks, or after truncate) is refused."""
        s = self._seq(sequence)
        if window < 1 or sinks < 0:
            raise InvalidInput(f"KvCache.evict: window ({window}) must be at least 1, sinks ({sinks}) not negative")
        ps, n = self.page_size, 0
        first = s.length - window + 1  # the first key that the next token sees
        for i, p in enumerate(s.pages):
            if p >= 0 and i * ps >= sinks and (i + 1) * ps <= first:
                self._drop(p)
                s.pages[i] = -1
                n += 1
        if n:
            s.evicted = True
            self._generation += 1
        return n

    def compact(self) -> int:
        """Move the pages in use to the front of the pools, so that every page
        from num_pages - free_pages() on is free.  Returns the pages moved."""
        live = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < live)
        high = [p for p in range(live, self.num_pages) if self._refs[p]]
        if not high:
            return 0
        moves = list(zip(high, holes))
        self._copy(moves)
        self._generation += 1
        to = dict(moves)
        for a, b in moves:
            self._refs[b], self._refs[a] = self._refs[a], 0
        for s in self._seqs.values():
            s.pages = [to.get(p, p) for p in s.pages]
        self._free = list(range(self.num_pages - 1, live - 1, -1))
        return len(moves)

    # -- helpers --------------------------------------------------------------------
    def _seq(self, sequence: int) -> _Sequence:
        s = self._seqs.get(sequence)
        if s is None:
            raise InvalidInput(f"KvCache: no sequence {sequence}")
        return s

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _drop(self, p: int) -> None:
        if p >= 0:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                self._free.append(p)

    def _cut(self, s: _Sequence, length: int) -> None:
        keep = -(-length // self.page_size)
        for p in s.pages[keep:]:
            self._drop(p)
        del s.pages[keep:]
        s.length = length

    def _own(self, *ts: Tensor) -> None:
        if any(t.device() is not self.device for t in ts):
            raise DeviceError("tensors live on different devices")

    def _check_step(self, op: str, step: KvStep, layer: int) -> None:
        if step._cache is not self:
            raise InvalidInput(f"{op}: the step belongs to another KvCache")
        if step._generation != self._generation:
            raise InvalidOperation(op, "the cache's pages have changed since the step was made")
        if not 0 <= layer < self.layers:
            raise InvalidInput(f"{op}: layer {layer} of {self.layers}")

    @staticmethod
    def _check_parents(items, parents) -> None:
        if len(parents) != len(items):
            raise InvalidInput(f"KvCache.batch: {len(parents)} trees for {len(items)} sequences")
        for (s, n), tree in zip(items, parents):
            if len(tree) != n or n > MAX_DRAFTS or any(not -1 <= p < j for j, p in enumerate(tree)):
                raise InvalidInput(f"KvCache.batch: the parents of sequence {s} must be {n} (at most {MAX_DRAFTS}), "
                                   "each -1 or below its draft")

    def _pages(self, step: KvStep, layer: int) -> N.KvPages:
        at = 4 * layer * self._layer
        return N.KvPages(self.k.ptr + at, self.v.ptr + at, self._layout, self._layout, self.num_pages, self.page_size,
                         self.kv_heads, self.head_dim, step._table, step._width)

    def _copy(self, moves: Sequence[tuple[int, int]]) -> None:
        """Pages copied, K and V, in every layer."""
        if not moves:
            return
        arr = C.c_int * len(moves)
        kv = N.KvPages(self.k.ptr, self.v.ptr, self._layout, self._layout, self.num_pages, self.page_size,
                       self.kv_heads, self.head_dim, None, 0)
        dev = self.device
        with dev._lock:
            dev.check(dev._lib.bch_kv_copy_pages(dev.ctx, kv, self.layers, self._layer, self._layer, len(moves),
                                                 arr(*[a for a, _ in moves]), arr(*[b for _, b in moves])),
                      "kv_copy_pages")

    def _own_pages(self, pages: Sequence[tuple[_Sequence, int]], more: int = 0) -> None:
        """Give each (sequence, page index) a page of its own: of the sequences
        that share one, all but the last (or all, if others hold it too) get a
        copy.  OutOfMemory, with nothing changed, unless that leaves `more` free."""
        refs: dict[int, int] = {}
        shared = []
        for s, i in pages:
            r = refs.get(s.pages[i], self._refs[s.pages[i]])
            if r > 1:
                refs[s.pages[i]] = r - 1
                shared.append((s, i))
        if len(shared) + more > len(self._free):
            raise OutOfMemory(f"KvCache: {len(shared) + more} pages needed, {len(self._free)} free")
        if not shared:
            return
        to = self._free[len(self._free) - len(shared):][::-1]
        self._copy([(s.pages[i], p) for (s, i), p in zip(shared, to)])
        self._generation += 1  # steps made before this name the shared pages
        for s, i in shared:
            self._refs[s.pages[i]] -= 1
            s.pages[i] = self._take()

    def _move(self, moves: Sequence[tuple[int, int, list[int]]]) -> None:
        """For each (sequence, to, positions): those keys to `to` on, the rest behind given up."""
        ps = self.page_size
        written = []
        for seq, to, positions in moves:
            if not positions or positions[-1] < to + len(positions):
                continue  # they are there already
            s = self._seqs[seq]
            pages = range(to // ps, -(-(to + len(positions)) // ps))
            if any(s.pages[i] < 0 for i in pages):
                raise InvalidOperation("KvCache", "a page that kept keys move into has been evicted")
            written += [(s, i) for i in pages]
        self._own_pages(written)
        moving = [(self._seqs[seq], to, positions) for seq, to, positions in moves if positions]
        if any(positions != list(range(to, to + len(positions))) for _, to, positions in moving):
            width = max(len(s.pages) for s, _, _ in moving)
            table = np.full((len(moving), width), -1, dtype=np.int32)
            for i, (s, _, _) in enumerate(moving):
                table[i, :len(s.pages)] = s.pages
            start = np.concatenate([[0], np.cumsum([len(p) for _, _, p in moving])])
            arrays = _I32(self.device, start, [x for _, _, p in moving for x in p], [to for _, to, _ in moving], table)
            starts, keep, tos, tables = arrays.ptrs
            dev = self.device
            self._generation += 1  # (not before: until here the step may be tried again)
            for b0 in range(0, len(moving), _KEEP_SEQUENCES):
                b1 = min(b0 + _KEEP_SEQUENCES, len(moving))
                for l0 in range(0, self.layers, _KEEP_LAYERS):
                    at = 4 * l0 * self._layer
                    kv = N.KvPages(self.k.ptr + at, self.v.ptr + at, self._layout, self._layout, self.num_pages,
                                   self.page_size, self.kv_heads, self.head_dim, tables + 4 * b0 * width, width)
                    with dev._lock:
                        dev.check(dev._lib.bch_kv_keep(dev.ctx, kv, min(_KEEP_LAYERS, self.layers - l0), self._layer,
                                                       self._layer, b1 - b0, int(start[b1]), C.c_void_p(starts + 4 * b0),
                                                       C.c_void_p(keep), C.c_void_p(tos + 4 * b0)), "kv_keep")
        self._generation += 1
        for seq, to, positions in moves:
            self._cut(self._seqs[seq], to + len(positions))
