"""8-bit integer linear layers over the C ABI: quantisation with one scale per
token or channel, the int8 product with its fused epilogue (scales, bias,
dropout, residual), the linear layer made of both with its backward pass, and
dropout whose mask is drawn again from (seed, stream_id, index) wherever it is
needed.

Torch tensors carry device memory and streams; all arithmetic runs in
libgemm_sm100a.so kernels, enqueued on the current stream of the tensors'
device.  Matrices are 2-D with unit stride along the last axis; int8 matrices
have a row stride that is a multiple of 16 bytes (as ``quantize_int8`` makes
them).  No call synchronises, and all of them can be captured into a CUDA graph
after one call outside of it.  They build no autograd graph: the backward pass
is ``linear_int8_backward``, and ``dropout`` itself for dropout.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import ERR_CANNOT_IMPLEMENT, GemmError, GemmInfo, OK, lib

TYPE_BF16, TYPE_FP16, TYPE_FP32 = 0, 1, 2
_TYPES = {torch.bfloat16: TYPE_BF16, torch.float16: TYPE_FP16, torch.float32: TYPE_FP32}
MAX_INT8_K = 131071   # 2^14 * k stays below 2^31


class DropoutArgs(C.Structure):
    _fields_ = [("p", C.c_double), ("seed", C.c_uint64), ("stream_id", C.c_uint64), ("seed_offset", C.c_void_p),
                ("row0", C.c_int64), ("col0", C.c_int64), ("row_elems", C.c_int64)]


class Int8GemmArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("d_type", C.c_int32),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("a", C.c_void_p), ("lda", C.c_int64),
        ("b", C.c_void_p), ("ldb", C.c_int64),
        ("d", C.c_void_p), ("ldd", C.c_int64),
        ("c", C.c_void_p), ("ldc", C.c_int64),
        ("scale_a", C.c_void_p), ("scale_b", C.c_void_p),
        ("bias", C.c_void_p), ("bias_type", C.c_int32),
        ("tile_n", C.c_int32), ("cta_group", C.c_int32), ("split_k", C.c_int32),
        ("drop", DropoutArgs),
        ("status", C.c_void_p), ("timeout_ms", C.c_uint32), ("flags", C.c_uint32),
    ]


class Int8QuantArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("x_type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("x", C.c_void_p), ("ldx", C.c_int64),
        ("q", C.c_void_p), ("ldq", C.c_int64),
        ("scale", C.c_void_p), ("col_sums", C.c_void_p),
        ("transpose", C.c_int32), ("reserved", C.c_int32),
        ("drop", DropoutArgs),
    ]


class Int8BackwardArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("type", C.c_int32),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("dy", C.c_void_p), ("lddy", C.c_int64),
        ("x", C.c_void_p), ("ldx", C.c_int64),
        ("wt", C.c_void_p), ("ldwt", C.c_int64),
        ("wt_scale", C.c_void_p),
        ("dx", C.c_void_p), ("lddx", C.c_int64),
        ("dw", C.c_void_p), ("lddw", C.c_int64),
        ("dbias", C.c_void_p), ("dw_type", C.c_int32), ("reserved", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64),
        ("drop", DropoutArgs),
        ("status", C.c_void_p),
    ]


class DropoutOpArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("type", C.c_int32),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("x", C.c_void_p), ("ldx", C.c_int64),
        ("residual", C.c_void_p), ("ldr", C.c_int64),
        ("y", C.c_void_p), ("ldy", C.c_int64),
        ("drop", DropoutArgs),
    ]


# The same layouts for struct.pack: one call fills an argument block several
# times faster than field by field, which counts for single tokens.
_DROP = "dQQPqqq"
_GEMM_PACK = struct.Struct("@IiqqqPqPqPqPqPPPiiii" + _DROP + "PII")
_QUANT_PACK = struct.Struct("@IiqqPqPqPPii" + _DROP)
_BACKWARD_PACK = struct.Struct("@IiqqqPqPqPqPPqPqPiiPq" + _DROP + "P")
_DROPOUT_PACK = struct.Struct("@IiqqPqPqPq" + _DROP)
_NO_DROP = (0.0, 0, 0, 0, 0, 0, 0)
_U64 = (1 << 64) - 1


class Dropout(NamedTuple):
    """Dropout with probability ``p`` of elements of a matrix with ``row_elems`` columns in
    all, of which the call sees the part that begins at (``row0``, ``col0``): the mask is a
    pure function of (seed, stream_id, (row0 + r) * row_elems + col0 + c), so a rank that owns a
    slice, and the backward pass, draw the same one again.

    ``seed``: an integer, or a CUDA tensor of one int64 that the kernel reads when it runs (so
    that replays of a captured graph draw new masks).  ``row_elems``: None = col0 + the columns
    of the call."""
    p: float
    seed: int | torch.Tensor = 0
    stream_id: int = 0
    row0: int = 0
    col0: int = 0
    row_elems: int | None = None


def _drop_fields(drop: Dropout | None, cols: int, index: int):
    if drop is None:
        return _NO_DROP
    p, seed, stream_id, row0, col0, row_elems = drop
    if p == 0.0:
        return _NO_DROP
    word = 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.get_device() != index:
            raise ValueError("a seed tensor holds one int64 on the operands' device")
        seed, word = 0, seed.data_ptr()
    return (p, seed & _U64, stream_id & _U64, word, row0, col0, col0 + cols if row_elems is None else row_elems)


def _matrix(t: torch.Tensor, name: str, dtype=None, shape=None, index: int | None = None) -> int:
    """Check one operand and return its row stride in elements.  `index`: the device it must be on."""
    try:
        (rows, cols), (ld, inner), dev = t.shape, t.stride(), t.get_device()
    except (AttributeError, ValueError):
        raise ValueError(f"{name} must be a 2-D tensor") from None
    if dev < 0 or (index is not None and dev != index):
        raise ValueError(f"{name} must be on the operands' CUDA device")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and (rows, cols) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {(rows, cols)}")
    if inner != 1 and cols > 1:
        raise ValueError(f"{name} must have unit stride along its last axis")
    if rows > 1:
        if ld < cols:
            raise ValueError(f"{name} has overlapping rows")
        return ld
    return cols or 1


def _floating(t: torch.Tensor, name: str) -> int:
    code = _TYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if code is None:
        raise ValueError(f"{name} must be a bfloat16, float16 or float32 tensor")
    return code


def _int8(t: torch.Tensor, name: str, shape=None, index: int | None = None) -> int:
    ld = _matrix(t, name, torch.int8, shape, index)
    if ld & 15 and t.shape[0] <= 1:
        ld = _pad16(ld)
    if ld & 15:
        raise ValueError(f"{name} must have a row stride that is a multiple of 16 bytes")
    return ld


def _vector(t: torch.Tensor, name: str, n: int, index: int, dtype=torch.float32) -> int:
    try:
        (size,), (step,), dev = t.shape, t.stride(), t.get_device()
    except (AttributeError, ValueError):
        size = -1
    if size != n or dev != index or (step != 1 and n > 1):
        raise ValueError(f"{name} must be a contiguous vector of {n} elements on the operands' device")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    return t.data_ptr()


def _pad16(n: int) -> int:
    return (n + 15) & ~15


# The current stream's handle; the Stream object that torch.cuda.current_stream builds costs
# 2 us, as much as a launch.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _row_bytes(cols: int) -> int:
    """Row stride of the int8 matrices made here: whole 128-byte lines, which a TMA row of an operand
    then never straddles (777 x 5000 x 2056: 11.4 us with rows of 2176 bytes, 18.8 with 2064)."""
    return (max(cols, 1) + 127) & ~127 if cols > 64 else _pad16(max(cols, 1))


def empty_int8(rows: int, cols: int, device) -> torch.Tensor:
    """An int8 matrix whose row stride is a multiple of 16 bytes (of 128 for more than 64 columns)."""
    return torch.empty_strided((rows, cols), (_row_bytes(cols), 1), dtype=torch.int8, device=device)


def quantize_int8(x: torch.Tensor, *, transpose: bool = False, dropout: Dropout | None = None,
                  column_sums: bool = False):
    """Symmetric int8 values and fp32 scales of ``x``: (q, scale) with one scale per row, or,
    with ``transpose``, one per column and ``q`` transposed.

    q = 127 x / max|x| rounded to the nearest integer (ties to even, decided exactly), scale =
    max|x| / 127; a row with NaN or Inf gets that as its scale.  ``dropout`` masks ``x`` first and
    puts 1 / (1 - p) into the scales.  ``column_sums`` (with ``transpose``) adds the fp32 sums of
    the masked columns: (q, scale, sums)."""
    code = _floating(x, "x")
    ldx = _matrix(x, "x")
    rows, cols = x.shape
    if column_sums and not transpose:
        raise ValueError("column_sums needs transpose=True")
    q = empty_int8(cols, rows, x.device) if transpose else empty_int8(rows, cols, x.device)
    scale = x.new_empty((cols if transpose else rows,), dtype=torch.float32)
    sums = x.new_empty((cols,), dtype=torch.float32) if column_sums else None
    if scale.shape[0]:
        if not transpose and cols == 0:
            raise ValueError("x has no columns")
        args = _QUANT_PACK.pack(_QUANT_PACK.size, code, rows, cols, x.data_ptr(), ldx, q.data_ptr(), q.stride(0),
                                scale.data_ptr(), 0 if sums is None else sums.data_ptr(), int(transpose), 0,
                                *_drop_fields(dropout, cols, x.get_device()))
        rc = lib().gemm_sm100a_quantize_int8(args, _raw_stream(x.get_device()))
        if rc != OK:
            raise GemmError(rc, "gemm_sm100a_quantize_int8")
    return (q, scale) if sums is None else (q, scale, sums)


def _output(out, m, n, dtype, like) -> torch.Tensor:
    if out is None:
        return like.new_empty((m, n), dtype=dtype)
    _matrix(out, "out", dtype, (m, n), like.get_device())
    return out


_KNOBS = {"tile_n", "cta_group", "split_k", "timeout_ms", "flags"}


def _tiles(knobs):
    if not _KNOBS.issuperset(knobs):
        raise TypeError(f"unknown knobs {sorted(set(knobs) - _KNOBS)}")
    return knobs.get("tile_n", 0), knobs.get("cta_group", 0), knobs.get("split_k", 0)


def _pack_gemm(index, code, m, n, k, a, lda, b, ldb, d, residual, a_scale, b_scale, bias, dropout, status, knobs):
    ldd = d.stride(0) if m > 1 else max(n, 1)
    c = ldc = 0
    if residual is not None:
        ldc = _matrix(residual, "residual", d.dtype, (m, n), index)
        c = residual.data_ptr()
    bias_ptr = bias_code = 0
    if bias is not None:
        bias_code = _floating(bias, "bias")
        bias_ptr = _vector(bias, "bias", n, index, None)
    return _GEMM_PACK.pack(_GEMM_PACK.size, code, m, n, k, a, lda, b, ldb, d.data_ptr(), ldd, c, ldc, a_scale, b_scale,
                           bias_ptr, bias_code, *(_tiles(knobs) if knobs else (0, 0, 0)),
                           *_drop_fields(dropout, n, index), 0 if status is None else status.data_ptr(),
                           knobs.get("timeout_ms", 0), knobs.get("flags", 0))


def _raise(rc, args, what):
    info = GemmInfo()
    lib().gemm_sm100a_int8_query(args, C.byref(info))
    raise GemmError(rc, f"{what} ({info.reason.decode()})")


def query_int8(args: Int8GemmArgs) -> tuple[int, GemmInfo]:
    """What ``gemm_sm100a_int8_launch`` would do with ``args`` (no launch)."""
    info = GemmInfo()
    return lib().gemm_sm100a_int8_query(bytes(args), C.byref(info)), info


def gemm_int8(a: torch.Tensor, a_scale: torch.Tensor | None, b: torch.Tensor, b_scale: torch.Tensor | None, *,
              bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
              dropout: Dropout | None = None, out_dtype: torch.dtype = torch.bfloat16,
              out: torch.Tensor | None = None, status: torch.Tensor | None = None, **knobs) -> torch.Tensor:
    """residual + dropout(a_scale[i] * b_scale[j] * (a . b^T) + bias[j]), (m, n), rounded once.

    ``a`` (m, k) and ``b`` (n, k) int8, ``a_scale`` (m) and ``b_scale`` (n) fp32 (None = 1);
    ``residual`` and ``out`` (which may be the residual) of ``out_dtype``.  The sum over k is
    exact, so the result does not depend on the batch or the tile.  ``status``: optional int32
    device word, as in ``gemm_into``.  Knobs: tile_n, cta_group, split_k, timeout_ms, flags."""
    lda = _int8(a, "a")
    index = a.get_device()
    m, k = a.shape
    ldb = _int8(b, "b", None, index)
    n, bk = b.shape
    if bk != k:
        raise ValueError(f"b must have {k} columns, as a has, got {bk}")
    if out is not None:
        out_dtype = out.dtype
    code = _TYPES.get(out_dtype)
    if code is None:
        raise ValueError("out_dtype must be bfloat16, float16 or float32")
    d = _output(out, m, n, out_dtype, a)
    sa = 0 if a_scale is None else _vector(a_scale, "a_scale", m, index)
    sb = 0 if b_scale is None else _vector(b_scale, "b_scale", n, index)
    args = _pack_gemm(index, code, m, n, k, a.data_ptr(), lda, b.data_ptr(), ldb, d, residual, sa, sb, bias, dropout,
                      status, knobs)
    rc = lib().gemm_sm100a_int8_launch(args, _raw_stream(index))
    if rc != OK:
        _raise(rc, args, "gemm_sm100a_int8_launch")
    return d


def linear_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, dropout: Dropout | None = None,
                out: torch.Tensor | None = None, status: torch.Tensor | None = None, **knobs) -> torch.Tensor:
    """x . w^T of floating tokens and int8 weights: ``quantize_int8(x)`` and ``gemm_int8`` with
    x's type as output, bit for bit, in one or two launches.

    ``x`` (m, k); ``w`` (n, k) int8 and ``w_scale`` (n) as ``quantize_int8`` makes them."""
    code = _floating(x, "x")
    ldx = _matrix(x, "x")
    index = x.get_device()
    m, k = x.shape
    ldw = _int8(w, "w", None, index)
    n, wk = w.shape
    if wk != k:
        raise ValueError(f"w must have {k} columns, as x has, got {wk}")
    sb = _vector(w_scale, "w_scale", n, index)
    d = x.new_empty((m, n)) if out is None else _output(out, m, n, x.dtype, x)
    lda = _row_bytes(k)
    q = sa = 0
    if m > 8 or knobs or m * k > 16384:   # else no workspace is needed
        work = x.new_empty((m * (lda + 4) + 16,), dtype=torch.uint8)          # int8 tokens, then their scales
        q = work.data_ptr()
        sa = q + m * lda
    args = _pack_gemm(index, code, m, n, k, q, lda, w.data_ptr(), ldw, d, residual, sa, sb, bias, dropout, status, knobs)
    rc = lib().gemm_sm100a_int8_linear(args, x.data_ptr(), code, ldx, _raw_stream(index))
    if rc != OK:
        _raise(rc, args, "gemm_sm100a_int8_linear")
    return d


def linear_int8_backward(dy: torch.Tensor, x: torch.Tensor, wt: torch.Tensor, wt_scale: torch.Tensor, *,
                         dropout: Dropout | None = None, dw_dtype: torch.dtype = torch.float32,
                         status: torch.Tensor | None = None):
    """Gradients (dx, dw, dbias) of y = residual + dropout(x . w^T + bias) for ``dy`` (m, n), by
    int8 products (the straight-through gradient of the quantised layer):

        dz = dropout(dy),  dx = dz . w,  dw = dz^T . x,  dbias = column sums of dz

    ``x`` (m, k) are the layer's tokens; ``wt`` (k, n) and ``wt_scale`` (k) are
    ``quantize_int8(w, transpose=True)``: the products contract over n and m, so the scales lie
    along the other axis.  dx has x's type, dw ``dw_dtype``, dbias is fp32.  The residual's
    gradient is dy.  m = 0 gives zeros for dw and dbias."""
    code = _floating(dy, "dy")
    lddy = _matrix(dy, "dy")
    index = dy.get_device()
    m, n = dy.shape
    _floating(x, "x")
    ldx = _matrix(x, "x", dy.dtype, None, index)
    xm, k = x.shape
    if xm != m:
        raise ValueError(f"x must have {m} rows, as dy has, got {xm}")
    dw_code = _TYPES.get(dw_dtype)
    if dw_code is None:
        raise ValueError("dw_dtype must be bfloat16, float16 or float32")
    ldwt = _int8(wt, "wt", (k, n), index)
    scale = _vector(wt_scale, "wt_scale", k, index)
    need = lib().gemm_sm100a_int8_backward_workspace(m, n, k)
    if need < 0:
        raise GemmError(ERR_CANNOT_IMPLEMENT, f"linear_int8_backward: sums over m and n are exact up to {MAX_INT8_K}")
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = x.new_empty((n, k), dtype=dw_dtype)
    dbias = x.new_empty((n,), dtype=torch.float32)
    work = x.new_empty((need,), dtype=torch.uint8)
    args = _BACKWARD_PACK.pack(_BACKWARD_PACK.size, code, m, n, k, dy.data_ptr(), lddy, x.data_ptr(), ldx, wt.data_ptr(),
                               ldwt, scale, dx.data_ptr(), k, dw.data_ptr(), k, dbias.data_ptr(), dw_code, 0,
                               work.data_ptr(), need, *_drop_fields(dropout, n, index),
                               0 if status is None else status.data_ptr())
    rc = lib().gemm_sm100a_int8_linear_backward(args, _raw_stream(index))
    if rc != OK:
        raise GemmError(rc, "gemm_sm100a_int8_linear_backward")
    return dx, dw, dbias


def dropout(x: torch.Tensor, drop: Dropout, *, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """residual + dropout(x), computed in fp32 and rounded once.  The gradient with respect to x
    is the same call on dy without the residual.  ``out`` may be x or residual."""
    code = _floating(x, "x")
    ldx = _matrix(x, "x")
    index = x.get_device()
    rows, cols = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if out is None else _output(out, rows, cols, x.dtype, x)
    ldy = y.stride(0) if rows > 1 else max(cols, 1)
    r = ldr = 0
    if residual is not None:
        ldr = _matrix(residual, "residual", x.dtype, (rows, cols), index)
        r = residual.data_ptr()
    args = _DROPOUT_PACK.pack(_DROPOUT_PACK.size, code, rows, cols, x.data_ptr(), ldx, r, ldr, y.data_ptr(), ldy,
                              *_drop_fields(drop, cols, index))
    rc = lib().gemm_sm100a_dropout(args, _raw_stream(index))
    if rc != OK:
        raise GemmError(rc, "gemm_sm100a_dropout")
    return y
