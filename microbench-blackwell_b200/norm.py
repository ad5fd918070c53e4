"""The residual stream around a block over the C ABI: the norm after the block, its gate and scale, the stream's
update and the norm before the next block in one kernel, their gradients in two, and the form whose result is the
4-bit operand of the next product.

    z = y * r(y) * post_weight        (y without post_weight)
    x_out = x + (gate * scale) * z    h = x_out * r(x_out) * weight     r(v) = 1 / sqrt(mean(v^2) + eps)

Matrices are 2-D with unit stride along the last axis, of one type (bf16, fp16 or fp32) and at most 16384 columns, on
one CUDA device; everything is enqueued on that device's current stream, nothing synchronises, and all calls can be
captured into a CUDA graph.  No autograd graph is built: the backward pass is ``residual_norm_backward``.  A refused
argument raises ValueError or GemmError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from .fp4 import Fp4
from .int8 import _host


class ResidualNormArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("x", C.c_void_p), ("ldx", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64),
        ("x_out", C.c_void_p), ("ldo", C.c_int64), ("h", C.c_void_p), ("ldh", C.c_int64),
        ("weight", C.c_void_p), ("post_weight", C.c_void_p), ("gate", C.c_void_p), ("ldg", C.c_int64),
        ("param_type", C.c_int32), ("block", C.c_int32), ("eps", C.c_double),
        ("scale", C.c_float), ("reserved", C.c_int32),
        ("values", C.c_void_p), ("ldv", C.c_int64), ("scales", C.c_void_p), ("row_scale", C.c_void_p),
    ]


class ResidualNormBackwardArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("dh", C.c_void_p), ("lddh", C.c_int64), ("dx_out", C.c_void_p), ("lddo", C.c_int64),
        ("x_out", C.c_void_p), ("ldo", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64),
        ("weight", C.c_void_p), ("post_weight", C.c_void_p), ("gate", C.c_void_p), ("ldg", C.c_int64),
        ("param_type", C.c_int32), ("scale", C.c_float), ("eps", C.c_double),
        ("dx", C.c_void_p), ("lddx", C.c_int64), ("dy", C.c_void_p), ("lddy", C.c_int64),
        ("dweight", C.c_void_p), ("dpost_weight", C.c_void_p), ("dgate", C.c_void_p), ("lddg", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64),
    ]


class NormGrads(NamedTuple):
    """Gradients of ``residual_norm``; None for what the call did not have."""
    dx: torch.Tensor
    dy: torch.Tensor | None
    dweight: torch.Tensor | None
    dpost_weight: torch.Tensor | None
    dgate: torch.Tensor | None


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, weight: torch.Tensor | None = None,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                  eps: float = 1e-6, fp4: int = 0, out: torch.Tensor | None = None):
    """(x_out, h): the residual stream ``x`` after a block's output ``y``, and its norm for the next block.

    ``post_weight``: the block's output is normed first.  ``gate``: a vector of columns, or a matrix like x with
    a row for each token.  ``weight``, ``post_weight`` and a vector gate have one type, x's or fp32.  Without ``y``,
    x_out is x.  ``fp4`` = 16 or 32: h is an ``Fp4`` with blocks of that size, from its fp32 values.  ``out`` takes
    x_out; it may be x or y.

    One fp32 operation follows the other from left to right, means of squares are taken in 64 bits; x_out is rounded to x's
    type, and h is that of the rounded x_out."""
    got = _host().residual_norm(x, y, weight, post_weight, gate, scale, eps, fp4, out)
    return (got[0], Fp4(got[1], got[2], got[3], x.shape[1], fp4)) if fp4 else got


def residual_norm_backward(dh: torch.Tensor, dx_out: torch.Tensor | None, x_out: torch.Tensor, y: torch.Tensor | None = None, *,
                           weight: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                           gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6) -> NormGrads:
    """Gradients of ``residual_norm`` for those of h and x_out (None: zero), from the call's x_out and arguments:

        g = dx_out + (gradient of h towards x_out),  dx = g,  dy = (gradient of (gate * scale) * z towards y for g)

    dx, dy and a matrix gate's dgate have x_out's type, dweight, dpost_weight and a vector gate's dgate are fp32 sums
    over the rows, in the same order for the same call.  No statistics are kept from the forward call; its row sums are fp32 here
    (of fp32 rows too), 64-bit in rows whose squares or products come near the ends of fp32's range."""
    return NormGrads(*_host().residual_norm_backward(dh, dx_out, x_out, y, weight, post_weight, gate, scale, eps))
