"""nn::fused_mlp over the GEMM's fused epilogue (bch_sgemm_ex).

Mirrors crates/barracuda/src/nn/fused_mlp.rs:
  Activation                                     fused_mlp.rs:25-31
  fused_mlp(input, weights, biases, activation)  fused_mlp.rs:38-168
with the same validation order and messages.  The reference records, per
layer, shaders/misc/linear_f64.wgsl (y = x W^T + b) and then
shaders/activation/relu_f64.wgsl over the layer's output, in one submit.
Here each layer is ONE launch: the GEMM adds the bias and applies ReLU in its
epilogue, so the output is written once and never re-read.

Weights may be [out, in] (the linear shader's layout, the product uses them
transposed) or [in, out] (used as they are).  For [in, out] weights that are
not square the reference still indexes the buffer as [out, in]
(linear_f64.wgsl:35 reads weight[out_f * in_features + in_f] whichever branch
of fused_mlp.rs:72-82 matched), which is not x W; this computes x W.
"""
from __future__ import annotations

import ctypes as C
import enum
from typing import Sequence

import numpy as np

from . import _native as N
from .error import InvalidInput, ShapeMismatch
from .tensor import HipDevice, Tensor, _Buffer, _check_i32, _same_device, get_device

__all__ = ["Activation", "fused_mlp", "linear", "Weights4", "linear4", "quantize4", "dequantize4"]


class Activation(enum.Enum):
    """fused_mlp.rs:25-31: the MLP's activation.  The reference has ReLU
    only; GELU (the tanh form of shaders/activation/gelu_f64.wgsl, the
    activation of transformer MLP blocks) is the same fused epilogue with
    BCH_ACT_GELU."""
    ReLU = "ReLU"
    GELU = "GELU"


def fused_mlp(input: Tensor, weights: Sequence[Tensor], biases: Sequence[Tensor],
              activation: Activation = Activation.ReLU) -> Tensor:
    if len(weights) != len(biases):
        raise InvalidInput(f"fused_mlp: weights len {len(weights)} != biases len {len(biases)}")
    if not weights:
        raise InvalidInput("fused_mlp: at least one layer required")
    shape = input.shape()
    if len(shape) != 2:
        raise InvalidInput(f"fused_mlp: input must be 2D, got {shape}")
    batch, in_features = shape
    layers = []  # (in, out, transb)
    for i, (w, b) in enumerate(zip(weights, biases)):
        ws = w.shape()
        if len(ws) != 2:
            raise InvalidInput(f"fused_mlp: weight[{i}] must be 2D")
        if ws[1] == in_features:
            out_f, in_f, transb = ws[0], ws[1], 1  # [out, in]: x W^T
        elif ws[0] == in_features:
            out_f, in_f, transb = ws[1], ws[0], 0  # [in, out]: x W
        else:
            raise InvalidInput(f"fused_mlp: weight[{i}] shape {ws} incompatible")
        if b.shape() != [out_f]:
            raise InvalidInput(f"fused_mlp: bias[{i}] shape mismatch")
        layers.append((in_f, out_f, transb))
        in_features = out_f
    dev = _same_device(input, *weights, *biases)
    act = {Activation.ReLU: N.BCH_ACT_RELU, Activation.GELU: N.BCH_ACT_GELU}[activation]
    x = input
    for (in_f, out_f, transb), w, b in zip(layers, weights, biases):
        _check_i32("fused_mlp", dev, batch=batch, in_features=in_f, out_features=out_f)
        y = Tensor.empty([batch, out_f], dev)
        if batch * out_f:
            with dev._lock:
                dev.check(dev._lib.bch_sgemm_ex(dev.ctx, transb, batch, out_f, in_f, C.c_void_p(x.ptr),
                                                max(in_f, 1), C.c_void_p(w.ptr),
                                                max(in_f if transb else out_f, 1), C.c_void_p(b.ptr), act,
                                                C.c_void_p(y.ptr), max(out_f, 1)), "fused_mlp")
        x = y
    return x


def linear(input: Tensor, weight: Tensor, bias: Tensor | None = None, activation: Activation | None = None) -> Tensor:
    """One layer of linear_f64.wgsl (y = x W^T + b, W [out, in]) with the
    activation that follows it fused into the GEMM's epilogue: one launch,
    the output written once.  input [batch, in]."""
    shape, ws = input.shape(), weight.shape()
    if len(shape) != 2 or len(ws) != 2 or ws[1] != shape[1]:
        raise InvalidInput(f"linear: input {shape} and weight {ws} (expected [out, {shape[-1] if shape else '?'}])")
    batch, in_f = shape
    out_f = ws[0]
    if bias is not None and bias.shape() != [out_f]:
        raise InvalidInput("linear: bias shape mismatch")
    dev = _same_device(input, weight, *([bias] if bias is not None else []))
    _check_i32("linear", dev, batch=batch, in_features=in_f, out_features=out_f)
    act = {None: N.BCH_ACT_NONE, Activation.ReLU: N.BCH_ACT_RELU, Activation.GELU: N.BCH_ACT_GELU}[activation]
    y = Tensor.empty([batch, out_f], dev)
    if batch * out_f:
        with dev._lock:
            dev.check(dev._lib.bch_sgemm_ex(dev.ctx, 1, batch, out_f, in_f, C.c_void_p(input.ptr), max(in_f, 1),
                                            C.c_void_p(weight.ptr), max(in_f, 1),
                                            C.c_void_p(bias.ptr) if bias is not None else None, act,
                                            C.c_void_p(y.ptr), max(out_f, 1)), "linear")
    return y


# ---- 4-bit weights: the reference's linear layer has f32 weights only; these stand beside it ----


def quantize4(weight, group: int = 128, zeros: bool = False):
    """(codes, scales, zeros or None) of weights [out, in], on the host: each group of `group` inputs of an output to
    the nearest of scale * (code - zero), code 0 .. 15.  Without zeros the zero point is 8 and codes are 1 .. 15; with
    them a group's codes span its values and 0."""
    w = np.asarray(weight, dtype=np.float32)
    if w.ndim != 2 or 0 in w.shape:
        raise InvalidInput(f"quantize4: weight {list(w.shape)} (expected [out, in])")
    if group < 32 or group % 32:
        raise InvalidInput(f"quantize4: groups of {group} inputs (needs a multiple of 32)")
    if not np.isfinite(w).all():
        raise InvalidInput("quantize4: weights must be finite")
    n, k = w.shape
    groups = -(-k // group)
    v = np.zeros((n, groups * group), np.float64)
    v[:, :k] = w
    v = v.reshape(n, groups, group)
    if zeros:
        lo, hi = np.minimum(v.min(2), 0.0), np.maximum(v.max(2), 0.0)
        scale = ((hi - lo) / 15.0).astype(np.float32)
    else:
        scale = (np.abs(v).max(2) / 7.0).astype(np.float32)
    s = np.where(scale > 0, scale, 1).astype(np.float64)
    zero = np.clip(np.rint(-lo / s), 0, 15) if zeros else np.full((n, groups), 8.0)
    code = np.clip(np.rint(v / s[:, :, None]) + zero[:, :, None], 0 if zeros else 1, 15).astype(np.uint8)
    code = code.reshape(n, -1)[:, :k + k % 2]
    if k % 2:
        code = np.concatenate([code, np.zeros((n, 1), np.uint8)], 1)[:, :k + 1]
        code[:, k] = 0
    return code[:, 0::2] | (code[:, 1::2] << 4), scale, zero.astype(np.uint8) if zeros else None


def dequantize4(codes, scales, group: int, k: int, zeros=None) -> np.ndarray:
    """The weights [out, k] that codes, scales and zeros stand for, on the host."""
    codes, scales = np.asarray(codes, dtype=np.uint8), np.asarray(scales, dtype=np.float32)
    code = np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)[:, :k].astype(np.float32)
    pick = np.arange(k) // group
    zero = np.float32(8) if zeros is None else np.asarray(zeros)[:, pick].astype(np.float32)
    return scales[:, pick] * (code - zero)


class Weights4:
    """A linear layer's weights [out, in] in 4 bits, in HBM in the layout that linear4's kernels read: codes [out,
    ceil(in / 2)] (two inputs a byte, the even one in the low half), scales and, unless they are 8, zeros [out,
    ceil(in / group)]; weight = scale * (code - zero)."""

    def __init__(self, codes, scales, in_features: int, group: int = 128, zeros=None, device: HipDevice | None = None):
        codes, scales = np.asarray(codes), np.ascontiguousarray(scales, dtype=np.float32)
        k = int(in_features)
        if codes.ndim != 2 or codes.dtype != np.uint8 or codes.shape[0] == 0 or k < 1 or codes.shape[1] != -(-k // 2):
            raise InvalidInput(f"Weights4: codes {list(codes.shape)} of {codes.dtype} (expected uint8 [out, {-(-k // 2)}])")
        if group < 32 or group % 32:
            raise InvalidInput(f"Weights4: groups of {group} inputs (needs a multiple of 32)")
        n = codes.shape[0]
        groups = [n, -(-k // group)]
        if list(scales.shape) != groups:
            raise ShapeMismatch(groups, list(scales.shape))
        if zeros is not None:
            zeros = np.asarray(zeros)
            if list(zeros.shape) != groups:
                raise ShapeMismatch(groups, list(zeros.shape))
            if zeros.dtype.kind not in "iu" or zeros.min() < 0 or zeros.max() > 15:
                raise InvalidInput("Weights4: zeros must be whole numbers from 0 to 15")
            zeros = np.ascontiguousarray(zeros, dtype=np.uint8)
        self.device = dev = device or get_device()
        group = min(group, -(-k // 32) * 32)  # one that covers all inputs is as good as any other
        _check_i32("Weights4", dev, out_features=n, in_features=k)
        self.out_features, self.in_features, self.group = n, k, group
        size = C.c_size_t()
        dev.check(dev._lib.bch_w4_bytes(n, k, group, C.byref(size)), "Weights4")
        self._buf = _Buffer(dev, size.value)
        parts = [np.ascontiguousarray(codes), scales] + ([zeros] if zeros is not None else [])
        bufs = [_Buffer(dev, p.nbytes) for p in parts]
        for b, p in zip(bufs, parts):
            dev.upload(b.ptr, p)
        with dev._lock:
            dev.check(dev._lib.bch_w4_pack(dev.ctx, n, k, group, C.c_void_p(bufs[0].ptr), codes.shape[1],
                                           C.c_void_p(bufs[1].ptr), C.c_void_p(bufs[2].ptr) if zeros is not None else None,
                                           C.c_void_p(self._buf.ptr)), "Weights4")
        self._w = N.W4(n, k, group, self._buf.ptr)

    @classmethod
    def quantize(cls, weight, group: int = 128, zeros: bool = False, device: HipDevice | None = None) -> "Weights4":
        """From f32 weights [out, in] (an array or a Tensor) by quantize4."""
        if isinstance(weight, Tensor):
            device = device or weight.device()
            weight = weight.to_numpy()
        codes, scales, z = quantize4(weight, group, zeros)
        return cls(codes, scales, np.shape(weight)[1], group, z, device)


def linear4(input: Tensor, weights: Weights4, bias: Tensor | None = None, activation: Activation | None = None) -> Tensor:
    """linear with 4-bit weights: act(x W^T + b), input [batch, in]; bias and activation in the product's own launch."""
    shape = input.shape()
    n, k = weights.out_features, weights.in_features
    if len(shape) != 2 or shape[1] != k:
        raise InvalidInput(f"linear4: input {shape} and weights [{n}, {k}]")
    if bias is not None and bias.shape() != [n]:
        raise InvalidInput("linear4: bias shape mismatch")
    dev = _same_device(input, Tensor(weights._buf, [0], weights.device), *([bias] if bias is not None else []))
    _check_i32("linear4", dev, batch=shape[0])
    act = {None: N.BCH_ACT_NONE, Activation.ReLU: N.BCH_ACT_RELU, Activation.GELU: N.BCH_ACT_GELU}[activation]
    y = Tensor.empty([shape[0], n], dev)
    if shape[0]:
        with dev._lock:
            dev.check(dev._lib.bch_w4_linear(dev.ctx, shape[0], weights._w, C.c_void_p(input.ptr), k,
                                             C.c_void_p(bias.ptr) if bias is not None else None, act, C.c_void_p(y.ptr), n),
                      "linear4")
    return y
