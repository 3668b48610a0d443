"""Sampling: a token for each row of logits, from given random numbers.

The reference ends at the softmax (ops/softmax.rs:31-144); this stands beside
it for programs that generate.  Of a row's tokens, weighing exp((x - max) /
temperature), the top_k largest logits stay (equal ones: the lower index
first), of these the shortest beginning that holds top_p of their weight, of
these the ones that weigh min_p of the largest or more; the token is the first
in index order whose cumulative weight exceeds u times the whole.

    out = logits.sample(u, Sampling(temperature=0.8, top_k=40, top_p=0.95))
    out.tokens()      # int32 [rows], on the host; out.ptr in HBM
    out.probs         # Tensor [rows]: each token's share of what it was drawn from
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Sequence

import numpy as np

from . import _native as N
from .error import InvalidInput, InvalidOperation, ShapeMismatch
from .tensor import Tensor, _Buffer, _I32_MAX, _check_i32, _same_device

__all__ = ["Sampling", "Sample", "Sampled"]


@dataclass(frozen=True)
class Sampling:
    """Temperature 0 takes the largest logit; top_k 0, top_p 1 and min_p 0 leave all tokens."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        if not (self.temperature >= 0 and self.top_k >= 0 and 0 <= self.top_p <= 1 and 0 <= self.min_p <= 1):
            raise InvalidInput(f"Sampling: temperature ({self.temperature}) and top_k ({self.top_k}) must not be negative, "
                               f"top_p ({self.top_p}) and min_p ({self.min_p}) from 0 to 1")
        if not np.isfinite(self.top_k) or self.top_k != int(self.top_k):
            raise InvalidInput(f"Sampling: top_k ({self.top_k}) must be a whole number")

    def _native(self) -> N.Sampling:
        return N.Sampling(self.temperature, min(int(self.top_k), _I32_MAX), self.top_p, self.min_p)


class Sampled:
    """The tokens chosen, int32 in HBM at `ptr`, and their probabilities."""

    def __init__(self, buffer: _Buffer, probs: Tensor):
        self._buf, self.probs = buffer, probs

    @property
    def ptr(self) -> int:
        return self._buf.ptr

    def tokens(self) -> np.ndarray:
        """Blocking readback; -1 for a row of nothing but -inf."""
        if self._buf.nbytes == 0:
            return np.empty(0, dtype=np.int32)
        return self._buf.device.download(self._buf.ptr, self._buf.nbytes).view(np.int32)


class Sample:
    """logits [rows, vocab], u [rows] (a Tensor, or numbers from 0 to below 1 that are uploaded), one rule for all
    rows or one for each."""

    def __init__(self, logits: Tensor, u, rule: Sampling | Sequence[Sampling] = Sampling()):
        shape = logits.shape()
        if len(shape) != 2:
            raise InvalidOperation("sample", f"requires 2D logits [rows, vocab], got {len(shape)}D")
        rows, vocab = shape
        if vocab == 0:
            raise InvalidOperation("sample", "no logits in a row")
        _check_i32("sample", logits.device(), rows=rows, vocab=vocab)
        if not isinstance(u, Tensor):
            u = np.asarray(u, dtype=np.float32)
            if list(u.shape) != [rows]:
                raise ShapeMismatch([rows], list(u.shape))
            if not np.all((u >= 0) & (u <= 1)):
                raise InvalidInput("sample: u must be numbers from 0 to below 1")
            u = Tensor.from_data(u, [rows], logits.device())
        elif u.shape() != [rows]:
            raise ShapeMismatch([rows], u.shape())
        if not isinstance(rule, Sampling):
            rule = list(rule)
            if len(rule) != rows or not all(isinstance(r, Sampling) for r in rule):
                raise InvalidInput(f"sample: {len(rule)} rules for {rows} rows")
        _same_device(logits, u)
        self.logits, self.u, self.rule = logits, u, rule

    def execute(self) -> Sampled:
        rows, vocab = self.logits.shape()
        dev = self.logits.device()
        out, probs = _Buffer(dev, 4 * rows), Tensor.empty([rows], dev)
        if rows == 0:
            return Sampled(out, probs)
        one, each = self.rule, None
        if not isinstance(one, Sampling):
            table = np.empty((rows, 4), np.float32)
            for i, r in enumerate(one):
                n = r._native()
                table[i] = n.temperature, 0, n.top_p, n.min_p
                table.view(np.int32)[i, 1] = n.top_k
            each, one = _Buffer(dev, table.nbytes), None
            dev.upload(each.ptr, table)
        with dev._lock:
            dev.check(dev._lib.bch_sample(dev.ctx, rows, vocab, C.c_void_p(self.logits.ptr), vocab,
                                          one._native() if one else None, C.c_void_p(each.ptr) if each else None,
                                          C.c_void_p(self.u.ptr), C.c_void_p(out.ptr), C.c_void_p(probs.ptr)), "sample")
        return Sampled(out, probs)
