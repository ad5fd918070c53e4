"""4-bit floating linear layers over the C ABI: quantisation to e2m1 values with a scale for each
block of 16 or 32 elements and one for each row, the product of such operands with its fused
epilogue, and the linear layer made of both.

Matrices are 2-D with unit stride along the last axis, on one CUDA device; everything is enqueued on that
device's current stream.  No call synchronises, and all of them can be captured into a CUDA graph.  They are
for serving: nothing here has a gradient.

Checks, allocations and the C-ABI calls are in csrc/torch_host.cpp, as those of the int8 operators.  A
refused argument raises ValueError or GemmError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import GemmInfo, lib
from .int8 import _NO_KNOBS, _host, _knob_values


class Fp4GemmArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("d_type", C.c_int32),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("a", C.c_void_p), ("lda", C.c_int64), ("a_scales", C.c_void_p), ("a_row_scale", C.c_void_p),
        ("b", C.c_void_p), ("ldb", C.c_int64), ("b_scales", C.c_void_p), ("b_row_scale", C.c_void_p),
        ("d", C.c_void_p), ("ldd", C.c_int64),
        ("c", C.c_void_p), ("ldc", C.c_int64),
        ("bias", C.c_void_p), ("bias_type", C.c_int32), ("block", C.c_int32),
        ("tile_n", C.c_int32), ("cta_group", C.c_int32), ("split_k", C.c_int32), ("reserved", C.c_int32),
        ("status", C.c_void_p), ("timeout_ms", C.c_uint32), ("flags", C.c_uint32),
    ]


class Fp4QuantArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("x_type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("x", C.c_void_p), ("ldx", C.c_int64),
        ("values", C.c_void_p), ("ldv", C.c_int64),
        ("scales", C.c_void_p), ("row_scale", C.c_void_p),
        ("block", C.c_int32), ("reserved", C.c_int32),
    ]


class Fp4DequantArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("y_type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("values", C.c_void_p), ("ldv", C.c_int64),
        ("scales", C.c_void_p), ("row_scale", C.c_void_p),
        ("y", C.c_void_p), ("ldy", C.c_int64),
        ("block", C.c_int32), ("reserved", C.c_int32),
    ]


class Fp4(NamedTuple):
    """A 4-bit matrix of ``values.shape[0]`` rows and ``cols`` columns; an element is value * block scale * row scale.

    ``values``: uint8 (rows, ceil(cols / 2)), two e2m1 codes to a byte, the even column in the low four bits,
    row stride a multiple of 16 bytes.  ``scales``: uint8, unsigned e4m3 for ``block`` 16 or e8m0 for 32, in
    tiles of 128 rows x 4 scales: that of row r and block column c at byte
    ((r // 128) * tiles + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4 with
    tiles = ceil(cols / 256) * 64 // block; those of columns beyond ``cols`` are not NaN.
    ``row_scale``: fp32 (rows), or None for 1."""
    values: torch.Tensor
    scales: torch.Tensor
    row_scale: torch.Tensor | None
    cols: int
    block: int


def fp4_scale_bytes(rows: int, cols: int, block: int) -> int:
    """Bytes of ``Fp4.scales``; -1 for sizes that are refused."""
    return lib().gemm_sm100a_fp4_scale_bytes(rows, cols, block)


def quantize_fp4(x: torch.Tensor, *, block: int = 16) -> Fp4:
    """The 4-bit form of the rows of ``x`` (bf16, fp16 or fp32):

    row scale g = 2^(floor(log2 max|x|) - 10), at least 2^-126; block scale s = the least e4m3 number
    (``block`` 16) or power of two from 2^-126 on (32) with 6 s >= max|x / g| over the block; values x / (g s) rounded to
    e2m1, ties to the even code, decided exactly.  A row with NaN or Inf gets that as its row scale.

    No element is clipped.  The conversion of the OCP microscaling formats takes 2^(floor(log2 max|x|) - 2) for blocks of 32
    instead and saturates what lies above 6 of it, so codes of its quantisers differ from these in blocks whose largest
    element is more than 1.5 times a power of two."""
    return Fp4(*_host().quantize_fp4(x, block), x.shape[1], block)


def dequantize_fp4(q: Fp4, *, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """What ``q`` stands for, computed in fp32 (where it is exact unless it leaves fp32's range) and rounded to ``dtype``."""
    return _host().dequantize_fp4(q, dtype, out)


def query_fp4(args: Fp4GemmArgs) -> tuple[int, GemmInfo]:
    """What ``gemm_sm100a_fp4_launch`` would do with ``args`` (no launch)."""
    info = GemmInfo()
    return lib().gemm_sm100a_fp4_query(bytes(args), C.byref(info)), info


def gemm_fp4(a: Fp4, b: Fp4, *, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
             status: torch.Tensor | None = None, **knobs) -> torch.Tensor:
    """residual + a . b^T + bias, (m, n), in bf16 or fp16: ``a`` (m, k) tokens, ``b`` (n, k) channels, of one block size.

    Products and block scales are exact, the sum is the tensor cores' fp32 (its order depends on the tile and the
    split), row scales, bias and residual fp32, rounded once.  ``residual`` and ``out`` of ``out_dtype``; ``out``
    is the residual or apart from it, and apart from the other operands.  ``status``: optional int32 device word,
    as in ``gemm_into``.  Knobs: tile_n, cta_group, split_k, timeout_ms, flags."""
    return _host().gemm_fp4(a, b, bias, residual, out_dtype, out, status, *(_knob_values(knobs) if knobs else _NO_KNOBS))


def linear_fp4(x: torch.Tensor, w: Fp4, *, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
               status: torch.Tensor | None = None, **knobs) -> torch.Tensor:
    """x . w^T of floating tokens and 4-bit weights: ``quantize_fp4(x)`` with w's block size and ``gemm_fp4``, in one
    or two launches.  The result has x's type (fp32 tokens need ``out_dtype``: bf16 or fp16).
    ``out`` (and ``residual`` with it) may be ``x``."""
    return _host().linear_fp4(x, w, bias, residual, out_dtype, out, status, *(_knob_values(knobs) if knobs else _NO_KNOBS))
