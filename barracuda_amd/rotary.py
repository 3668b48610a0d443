"""Rotary positions: pairs of a head's columns turned by an angle that grows with the row's position.

The reference has no positional op; these stand beside its attention
(ops/causal_attn/mod.rs:64-158) for programs whose models place tokens this
way.  The pair i of a row at position p is turned by p * freq[i], freq[i] =
base^(-2i/dim), and a long context slows the pairs down (`scaling`):

    linear   all of them by `factor`
    base     a larger base: the slowest pair by `factor`, the fastest not at all
    parts    each by itself: pairs that turn `fast` times or more within the
             `context` that the model was trained on stay, those that turn
             `slow` times or less are slowed by `factor`, the others in between

    rotary = Rotary(128)
    q, k = q.rotary(rotary), k.rotary(rotary)          # [B, H, S, D]
    dq = dq.rotary(rotary, inverse=True)               # the gradient's way back
    q = cache.append_rotary(step, layer, rotary, q, k, v)
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Sequence

import numpy as np

from . import _native as N
from .error import InvalidInput, InvalidOperation, ShapeMismatch
from .kv_cache import _I32
from .tensor import HipDevice, Tensor, _Buffer, _check_i32, _dense, _numel, _same_device, get_device

__all__ = ["Rotary", "RotaryPositions", "rotary_freqs"]

_FASTEST = 2.0**19  # radians a position: angles of 32-bit positions stay below 2^50, where 64 bits still tell their turns
_SCALINGS = ("none", "linear", "base", "parts")


def rotary_freqs(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, context: float = 0.0,
                 fast: float = 32.0, slow: float = 1.0) -> np.ndarray:
    """Radians a position of each of dim/2 pairs, float64."""
    if dim < 2 or dim % 2:
        raise InvalidInput(f"rotary: {dim} columns to turn (needs an even number from 2 on)")
    if scaling not in _SCALINGS:
        raise InvalidInput(f"rotary: scaling {scaling!r} is none of {', '.join(_SCALINGS)}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise InvalidInput(f"rotary: base ({base}) and factor ({factor}) must be positive")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = float(base) ** (-2.0 * np.arange(dim // 2, dtype=np.float64) / dim)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        if not (context > 0 and fast > slow):
            raise InvalidInput(f"rotary: parts need a context ({context}) and fast ({fast}) above slow ({slow})")
        stay = np.clip((context * f / (2.0 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        f = f * (stay + (1.0 - stay) / factor)
    return f


class Rotary:
    """What a model turns its heads by: of head_dim columns the first `dim` (all
    of them unless given), column i with i + dim/2 or (interleaved) 2i with
    2i + 1, results times `scale`.  freqs, if given, are radians a position of
    each pair instead of what base and scaling (rotary_freqs) say."""

    def __init__(self, head_dim: int, dim: int | None = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", factor: float = 1.0, context: float = 0.0, fast: float = 32.0, slow: float = 1.0,
                 scale: float = 1.0, freqs: Sequence[float] | None = None, device: HipDevice | None = None):
        dim = head_dim if dim is None else dim
        if dim > head_dim:
            raise InvalidInput(f"rotary: {dim} columns to turn of a head of {head_dim}")
        f = rotary_freqs(dim, base, scaling, factor, context, fast, slow)
        if freqs is not None:
            f = np.ascontiguousarray(freqs, dtype=np.float64).reshape(-1)
            if f.size != dim // 2:
                raise ShapeMismatch([dim // 2], [f.size])
        if not np.all(np.abs(f) <= _FASTEST):
            raise InvalidInput(f"rotary: radians a position must be numbers of at most {_FASTEST:g}")
        self.head_dim, self.dim, self.interleaved, self.scale = int(head_dim), int(dim), bool(interleaved), float(scale)
        self.freqs = f
        self.device = device or get_device()
        self._buf = _Buffer(self.device, f.nbytes)
        self.device.upload(self._buf.ptr, f)
        self._plan = N.Rotary(self.dim, int(self.interleaved), self.scale, self._buf.ptr)


class RotaryPositions:
    """x turned by its rows' positions: x [B, H, S, D] (heads_last: [B, S, H, D]), row i of batch b
    at positions[b][i], or at first + i.  inverse turns back: what the
    gradient of the result gives for x."""

    def __init__(self, input: Tensor, rotary: Rotary, first: int = 0, positions=None, inverse: bool = False,
                 heads_last: bool = False):
        shape = input.shape()
        if len(shape) != 4:
            raise InvalidOperation("rotary", f"requires a 4D tensor, got {len(shape)}D")
        if shape[3] != rotary.head_dim:
            raise ShapeMismatch([rotary.head_dim], shape)
        self.b, self.d = shape[0], shape[3]
        self.s, self.h = (shape[1], shape[2]) if heads_last else (shape[2], shape[1])
        if positions is not None:
            positions = np.asarray(positions)
            if list(positions.shape) != [self.b, self.s]:
                raise ShapeMismatch([self.b, self.s], list(positions.shape))
            if positions.size and (positions.dtype.kind not in "iu" or positions.min() < -2**31 or positions.max() >= 2**31):
                raise InvalidInput("rotary: positions must be whole numbers of 32 bits")
        elif abs(int(first)) >= 2**31:
            raise InvalidInput(f"rotary: first ({first}) must fit 32 bits")
        if rotary.device is not input.device():
            _same_device(input, Tensor(rotary._buf, [0], rotary.device))
        self.input, self.rotary, self.first, self.positions = input, rotary, int(first), positions
        self.inverse, self.heads_last = bool(inverse), bool(heads_last)

    def execute(self) -> Tensor:
        dev, b, h, s, d = self.input.device(), self.b, self.h, self.s, self.d
        _check_i32("rotary", dev, batch=b, heads=h, rows=s, head_dim=d)
        out = Tensor.empty(self.input.shape(), dev)
        if _numel(self.input.shape()) == 0:
            return out
        lay = N.AttnLayout(s * h * d, d, h * d) if self.heads_last else _dense(h, s, d)
        pos = None if self.positions is None else _I32(dev, self.positions)
        with dev._lock:
            dev.check(dev._lib.bch_rotary(dev.ctx, b, h, s, d, self.rotary._plan, int(self.inverse), self.first,
                                          C.c_void_p(pos.ptrs[0]) if pos else None, C.c_void_p(self.input.ptr), lay,
                                          C.c_void_p(out.ptr), lay), "rotary")
        return out
