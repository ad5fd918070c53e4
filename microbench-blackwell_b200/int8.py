"""8-bit integer linear layers over the C ABI: quantisation with one scale per
token or channel, the int8 product with its fused epilogue (scales, bias,
dropout, residual), the linear layer made of both with its backward pass, and
dropout whose mask is drawn again from (seed, stream_id, index) wherever it is
needed.

Torch tensors carry device memory and streams; all arithmetic runs in
libgemm_sm100a.so kernels, enqueued on the current stream of the tensors'
device.  Matrices are 2-D with unit stride along the last axis; int8 matrices
have a row stride that is a multiple of 16 bytes (as ``quantize_int8`` makes
them).  No call synchronises, and all of them can be captured into a CUDA graph.
They build no autograd graph: the backward pass is ``linear_int8_backward``, and
``dropout`` itself for dropout.

Checks, allocations and the C-ABI calls are in csrc/torch_host.cpp (built into
lib/gemm_sm100a_torch.so): a small call is bound by the host.  A refused argument
raises ValueError or GemmError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from typing import NamedTuple

import torch

from . import GemmError, GemmInfo, PKG_DIR, lib

TORCH_LIB_PATH = PKG_DIR / "lib" / "gemm_sm100a_torch.so"
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


_host_module = None


def _raise_gemm_error(code: int, what: str):
    raise GemmError(code, what)


def _host():
    """The extension module (raises if it was not built: no fallback path exists)."""
    global _host_module
    if _host_module is None:
        lib()
        if not TORCH_LIB_PATH.exists():
            raise RuntimeError(f"{TORCH_LIB_PATH} is missing: build it with `make -C {PKG_DIR}` "
                               "(or __graft_entry__.build()); there is no CPU fallback")
        loader = importlib.machinery.ExtensionFileLoader("gemm_sm100a_torch", str(TORCH_LIB_PATH))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("gemm_sm100a_torch", loader))
        loader.exec_module(module)
        module.set_raise(_raise_gemm_error)
        _host_module = module
    return _host_module


_KNOBS = {"tile_n", "cta_group", "split_k", "timeout_ms", "flags"}
_NO_KNOBS = (0, 0, 0, 0, 0)


def _knob_values(knobs):
    if not _KNOBS.issuperset(knobs):
        raise TypeError(f"unknown knobs {sorted(set(knobs) - _KNOBS)}")
    return tuple(knobs.get(k, 0) for k in ("tile_n", "cta_group", "split_k", "timeout_ms", "flags"))


def empty_int8(rows: int, cols: int, device) -> torch.Tensor:
    """An int8 matrix whose row stride is a multiple of 16 bytes (of 128 for more than 64 columns)."""
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"an int8 matrix for these operators is on a CUDA device, not on {device}")
    index = torch.cuda.current_device() if device.index is None else device.index
    return _host().empty(rows, cols, index)


def quantize_int8(x: torch.Tensor, *, transpose: bool = False, dropout: Dropout | None = None,
                  column_sums: bool = False):
    """Symmetric int8 values and fp32 scales of ``x``: (q, scale) with one scale per row, or,
    with ``transpose``, one per column and ``q`` transposed.

    q = 127 x / max|x| rounded to the nearest integer (ties to even, decided exactly), scale =
    max|x| / 127; a row with NaN or Inf gets that as its scale.  ``dropout`` masks ``x`` first and
    puts 1 / (1 - p) into the scales.  ``column_sums`` (with ``transpose``) adds the fp32 sums of
    the masked columns: (q, scale, sums)."""
    return _host().quantize(x, transpose, dropout, column_sums)


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
    ``residual`` and ``out`` of ``out_dtype``; ``out`` is the residual or apart from it, and apart
    from the other operands.  The sum over k is exact, so the result does not depend on the batch or
    the tile.  ``status``: optional int32 device word, as in ``gemm_into``.  Knobs: tile_n, cta_group,
    split_k, timeout_ms, flags."""
    return _host().gemm(a, a_scale, b, b_scale, bias, residual, dropout, out_dtype, out, status,
                        *(_knob_values(knobs) if knobs else _NO_KNOBS))


def linear_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, dropout: Dropout | None = None,
                out: torch.Tensor | None = None, status: torch.Tensor | None = None, **knobs) -> torch.Tensor:
    """x . w^T of floating tokens and int8 weights: ``quantize_int8(x)`` and ``gemm_int8`` with
    x's type as output, bit for bit, in one or two launches.  ``out`` (and ``residual`` with it) may
    be ``x``.

    ``x`` (m, k); ``w`` (n, k) int8 and ``w_scale`` (n) as ``quantize_int8`` makes them."""
    return _host().linear(x, w, w_scale, bias, residual, dropout, out, status,
                          *(_knob_values(knobs) if knobs else _NO_KNOBS))


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
    return _host().backward(dy, x, wt, wt_scale, dropout, dw_dtype, status)


def dropout(x: torch.Tensor, drop: Dropout, *, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """residual + dropout(x), computed in fp32 and rounded once.  The gradient with respect to x
    is the same call on dy without the residual.  ``out`` may be x or residual; another overlap is
    refused."""
    return _host().dropout(x, drop, residual, out)
