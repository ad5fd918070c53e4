// torch_host.cpp -- the host side of the int8 and 4-bit operators and the norms for PyTorch callers:
// argument checks, output and workspace allocation, and the C-ABI call, as one
// CPython extension.  A small call is bound by the host, and in Python its
// checks, allocations and argument packing took twice as long as the launch.
// The functions take positional arguments only; int8.py, fp4.py and norm.py give them
// their signatures and documentation.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

#include "gemm_sm100a.h"

namespace {

PyObject* g_raise = nullptr;   // (code, what): raises GemmError

// A check that failed: the message is in the Python error already.
struct Refused {};

template <typename... A>
[[noreturn]] void refuse(const char* fmt, A... a) {
  PyErr_Format(PyExc_ValueError, fmt, a...);
  throw Refused();
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return GEMM_TYPE_BF16;
    case at::kHalf: return GEMM_TYPE_FP16;
    case at::kFloat: return GEMM_TYPE_FP32;
    default: return -1;
  }
}

int64_t pad16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Row stride of the int8 matrices made here: whole 128-byte lines, which a TMA row of an operand then never
// straddles (777 x 5000 x 2056: 12.5 us with rows of 2176 bytes, 19.8 with 2064).
int64_t row_bytes(int64_t cols) {
  if (cols < 1) cols = 1;
  return cols > 64 ? (cols + 127) & ~(int64_t)127 : pad16(cols);
}

struct Matrix {
  const at::Tensor* t;
  int64_t rows, cols, ld;
  void* ptr;
  at::ScalarType dtype;
  int index;
};

const at::Tensor& tensor(PyObject* o, const char* name, int dims) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.dim() == dims && t.layout() == c10::kStrided) return t;
  }
  if (dims == 2) refuse("%s must be a 2-D tensor", name);
  refuse("%s must be a vector", name);
}

// A 2-D operand on device `index` (-1: any CUDA device).
Matrix matrix(PyObject* o, const char* name, int index) {
  const at::Tensor& t = tensor(o, name, 2);
  if (!t.is_cuda() || (index >= 0 && t.get_device() != index)) refuse("%s must be on the operands' CUDA device", name);
  Matrix m;
  m.t = &t;
  m.rows = t.size(0);
  m.cols = t.size(1);
  m.ld = t.stride(0);
  m.dtype = t.scalar_type();
  m.index = t.get_device();
  if (t.stride(1) != 1 && m.cols > 1) refuse("%s must have unit stride along its last axis", name);
  if (m.rows > 1) {
    if (m.ld < m.cols) refuse("%s has overlapping rows", name);
  } else {
    m.ld = m.cols > 0 ? m.cols : 1;
  }
  m.ptr = t.data_ptr();
  return m;
}

int floating(const Matrix& m, const char* name) {
  const int code = type_code(m.dtype);
  if (code < 0) refuse("%s must be a bfloat16, float16 or float32 tensor", name);
  return code;
}

void shape(const Matrix& m, const char* name, int64_t rows, int64_t cols) {
  if (m.rows != rows || m.cols != cols)
    refuse("%s must have shape (%lld, %lld), got (%lld, %lld)", name, (long long)rows, (long long)cols, (long long)m.rows,
           (long long)m.cols);
}

void same_type(const Matrix& m, const char* name, at::ScalarType t) {
  if (m.dtype != t) refuse("%s must be %s, got %s", name, c10::toString(t), c10::toString(m.dtype));
}

Matrix int8_matrix(PyObject* o, const char* name, int index) {
  Matrix m = matrix(o, name, index);
  same_type(m, name, at::kChar);
  if (m.rows <= 1) m.ld = pad16(m.ld);
  if (m.ld & 15) refuse("%s must have a row stride that is a multiple of 16 bytes", name);
  return m;
}

// A contiguous vector of n elements; its type in `code` (of the three) or, with code NULL, fp32.
const void* vector(PyObject* o, const char* name, int64_t n, int index, int32_t* code) {
  const at::Tensor& t = tensor(o, name, 1);
  if (t.size(0) != n || !t.is_cuda() || t.get_device() != index || (t.stride(0) != 1 && n > 1))
    refuse("%s must be a contiguous vector of %lld elements on the operands' device", name, (long long)n);
  const int c = type_code(t.scalar_type());
  if (code) {
    if (c < 0) refuse("%s must be a bfloat16, float16 or float32 tensor", name);
    *code = c;
  } else if (c != GEMM_TYPE_FP32) {
    refuse("%s must be float32", name);
  }
  return t.data_ptr();
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused();
  return v;
}

int32_t knob(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < 0 || v > INT32_MAX) refuse("%s must be between 0 and 2^31 - 1", name);
  return (int32_t)v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v == 1;
}

// A Dropout tuple (p, seed, stream_id, row0, col0, row_elems) or None.
DropoutArgs dropout_args(PyObject* o, int64_t cols, int index) {
  DropoutArgs d;
  memset(&d, 0, sizeof(d));
  if (o == Py_None) return d;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 6) refuse("dropout must be a Dropout");
  d.p = PyFloat_AsDouble(PyTuple_GET_ITEM(o, 0));
  if (d.p == -1.0 && PyErr_Occurred()) throw Refused();
  if (d.p == 0.0) return d;
  PyObject* const seed = PyTuple_GET_ITEM(o, 1);
  if (THPVariable_Check(seed)) {
    const at::Tensor& t = THPVariable_Unpack(seed);
    if (t.scalar_type() != at::kLong || t.numel() != 1 || !t.is_cuda() || t.get_device() != index)
      refuse("a seed tensor holds one int64 on the operands' device");
    d.seed_offset = static_cast<const uint64_t*>(t.data_ptr());
  } else {
    d.seed = PyLong_AsUnsignedLongLongMask(seed);
  }
  d.stream_id = PyLong_AsUnsignedLongLongMask(PyTuple_GET_ITEM(o, 2));
  if (PyErr_Occurred()) throw Refused();
  d.row0 = integer(PyTuple_GET_ITEM(o, 3));
  d.col0 = integer(PyTuple_GET_ITEM(o, 4));
  PyObject* const row_elems = PyTuple_GET_ITEM(o, 5);
  d.row_elems = row_elems == Py_None ? d.col0 + cols : integer(row_elems);
  return d;
}

at::ScalarType dtype_arg(PyObject* o, const char* name) {
  if (THPDtype_Check(o)) {
    const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
    if (type_code(t) >= 0) return t;
  }
  refuse("%s must be bfloat16, float16 or float32", name);
}

int32_t* status_word(PyObject* o, int index) {
  if (o == Py_None) return nullptr;
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() == at::kInt && t.numel() == 1 && t.is_cuda() && t.get_device() == index)
      return static_cast<int32_t*>(t.data_ptr());
  }
  refuse("status holds one int32 on the operands' device");
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType t, int index) {
  return at::Tensor(at::detail::empty_cuda(size, t, at::Device(at::kCUDA, (c10::DeviceIndex)index), std::nullopt));
}

// An int8 matrix whose row stride is row_bytes(cols).
at::Tensor empty_int8(int64_t rows, int64_t cols, int index) {
  return at::Tensor(at::detail::empty_strided_cuda({rows, cols}, {row_bytes(cols), 1}, at::kChar,
                                                   at::Device(at::kCUDA, (c10::DeviceIndex)index)));
}

void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }

[[noreturn]] void failed(int rc, const char* what, const char* reason) {
  char text[256];
  snprintf(text, sizeof(text), reason && *reason ? "%s (%s)" : "%s", what, reason);
  PyObject* const r = PyObject_CallFunction(g_raise, "is", rc, text);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, text);
  throw Refused();
}

// The output of a product or of dropout: `o`, or a new packed one.
struct Output {
  at::Tensor fresh;
  PyObject* given = nullptr;
  bool written = false;      // `given` is (or is about to be) overwritten
  void* ptr;
  int64_t ld;
  // After the launch.  Autograd then sees that a tensor which it has saved is no longer what it was.
  PyObject* wrap() {
    if (given) {
      if (written) {
        const at::Tensor& t = THPVariable_Unpack(given);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
      }
      Py_INCREF(given);
      return given;
    }
    return THPVariable_Wrap(std::move(fresh));
  }
};

Output output(PyObject* o, int64_t rows, int64_t cols, at::ScalarType t, int index) {
  Output out;
  if (o != Py_None) {
    const Matrix m = matrix(o, "out", index);
    same_type(m, "out", t);
    shape(m, "out", rows, cols);
    out.given = o;
    out.written = true;
    out.ptr = m.ptr;
    out.ld = m.ld;
  } else {
    out.fresh = empty({rows, cols}, t, index);
    out.ptr = out.fresh.data_ptr();
    out.ld = cols > 0 ? cols : 1;
  }
  return out;
}

template <typename F>
PyObject* guarded(F&& body) {
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* const torch = PyImport_ImportModule("torch");
    PyObject* const type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
    return nullptr;
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    throw Refused();
  }
}

// The part of Int8GemmArgs that products and linear layers share; args: bias, residual, dropout,
// status, tile_n, cta_group, split_k, timeout_ms, flags.
void common(Int8GemmArgs& g, PyObject* bias, PyObject* residual, PyObject* drop, PyObject* status, PyObject* const* knobs,
            at::ScalarType t, int index) {
  g.struct_size = sizeof(g);
  g.d_type = type_code(t);
  if (residual != Py_None) {
    const Matrix c = matrix(residual, "residual", index);
    same_type(c, "residual", t);
    shape(c, "residual", g.m, g.n);
    g.c = c.ptr;
    g.ldc = c.ld;
  }
  if (bias != Py_None) g.bias = vector(bias, "bias", g.n, index, &g.bias_type);
  g.drop = dropout_args(drop, g.n, index);
  g.status = status_word(status, index);
  g.tile_n = knob(knobs[0], "tile_n");
  g.cta_group = knob(knobs[1], "cta_group");
  g.split_k = knob(knobs[2], "split_k");
  g.timeout_ms = (uint32_t)knob(knobs[3], "timeout_ms");
  g.flags = (uint32_t)knob(knobs[4], "flags");
}

[[noreturn]] void failed_product(int rc, const Int8GemmArgs& g, const char* what) {
  GemmInfo info;
  gemm_sm100a_int8_query(&g, &info);
  failed(rc, what, info.reason);
}

// (a, a_scale, b, b_scale, bias, residual, dropout, out_dtype, out, status, tile_n, cta_group, split_k, timeout_ms, flags)
PyObject* py_gemm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 15);
    const Matrix a = int8_matrix(v[0], "a", -1), b = int8_matrix(v[2], "b", a.index);
    if (b.cols != a.cols) refuse("b must have %lld columns, as a has, got %lld", (long long)a.cols, (long long)b.cols);
    Int8GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.m = a.rows; g.n = b.rows; g.k = a.cols;
    at::ScalarType t;
    if (v[8] != Py_None) {
      const Matrix d = matrix(v[8], "out", a.index);
      floating(d, "out");
      t = d.dtype;
    } else {
      t = dtype_arg(v[7], "out_dtype");
    }
    if (v[1] != Py_None) g.scale_a = static_cast<const float*>(vector(v[1], "a_scale", g.m, a.index, nullptr));
    if (v[3] != Py_None) g.scale_b = static_cast<const float*>(vector(v[3], "b_scale", g.n, a.index, nullptr));
    common(g, v[4], v[5], v[6], v[9], v + 10, t, a.index);
    Output d = output(v[8], g.m, g.n, t, a.index);
    g.a = a.ptr; g.lda = a.ld; g.b = b.ptr; g.ldb = b.ld; g.d = d.ptr; g.ldd = d.ld;
    const int rc = gemm_sm100a_int8_launch(&g, stream_of(a.index));
    if (rc != GEMM_OK) failed_product(rc, g, "gemm_sm100a_int8_launch");
    return d.wrap();
  });
}

// (x, w, w_scale, bias, residual, dropout, out, status, tile_n, cta_group, split_k, timeout_ms, flags)
PyObject* py_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 13);
    const Matrix x = matrix(v[0], "x", -1);
    const int code = floating(x, "x");
    const Matrix w = int8_matrix(v[1], "w", x.index);
    if (w.cols != x.cols) refuse("w must have %lld columns, as x has, got %lld", (long long)x.cols, (long long)w.cols);
    Int8GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.m = x.rows; g.n = w.rows; g.k = x.cols;
    g.scale_b = static_cast<const float*>(vector(v[2], "w_scale", g.n, x.index, nullptr));
    common(g, v[3], v[4], v[5], v[7], v + 8, x.dtype, x.index);
    Output d = output(v[6], g.m, g.n, x.dtype, x.index);
    g.lda = row_bytes(g.k);
    at::Tensor work;
    const uint8_t* const x0 = static_cast<const uint8_t*>(x.ptr);
    const uint8_t* const d0 = static_cast<const uint8_t*>(d.ptr);
    const int64_t e = (int64_t)x.t->element_size();
    const bool over = d.given && g.m > 0 && x0 < d0 + ((g.m - 1) * d.ld + g.n) * e && d0 < x0 + ((g.m - 1) * x.ld + g.k) * e;
    if (g.m > 8 || g.m * g.k > 16384 || g.tile_n || g.cta_group || g.split_k || g.flags || over) {   // else no workspace is needed
      work = empty({g.m * (g.lda + 4) + 16}, at::kByte, x.index);                            // int8 tokens, then their scales
      uint8_t* const q = static_cast<uint8_t*>(work.data_ptr());
      g.a = q;
      g.scale_a = reinterpret_cast<const float*>(q + g.m * g.lda);
    }
    g.b = w.ptr; g.ldb = w.ld; g.d = d.ptr; g.ldd = d.ld;
    const int rc = gemm_sm100a_int8_linear(&g, x.ptr, code, x.ld, stream_of(x.index));
    if (rc != GEMM_OK) {
      if (!g.a) g.a = g.b;   // for the reason only: without a workspace the query would name its absence
      failed_product(rc, g, "gemm_sm100a_int8_linear");
    }
    return d.wrap();
  });
}

// (dy, x, wt, wt_scale, dropout, dw_dtype, status) -> (dx, dw, dbias)
PyObject* py_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 7);
    const Matrix dy = matrix(v[0], "dy", -1);
    const int code = floating(dy, "dy");
    const Matrix x = matrix(v[1], "x", dy.index);
    same_type(x, "x", dy.dtype);
    if (x.rows != dy.rows) refuse("x must have %lld rows, as dy has, got %lld", (long long)dy.rows, (long long)x.rows);
    const Matrix wt = int8_matrix(v[2], "wt", dy.index);
    shape(wt, "wt", x.cols, dy.cols);
    Int8BackwardArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.type = code;
    g.m = dy.rows; g.n = dy.cols; g.k = x.cols;
    g.wt_scale = static_cast<const float*>(vector(v[3], "wt_scale", g.k, dy.index, nullptr));
    g.drop = dropout_args(v[4], g.n, dy.index);
    const at::ScalarType dw_type = dtype_arg(v[5], "dw_dtype");
    g.dw_type = type_code(dw_type);
    g.status = status_word(v[6], dy.index);
    g.workspace_bytes = gemm_sm100a_int8_backward_workspace(g.m, g.n, g.k);
    if (g.workspace_bytes < 0)
      failed(GEMM_ERR_CANNOT_IMPLEMENT, "gemm_sm100a_int8_linear_backward", "sums over m and n are exact up to 131071");
    at::Tensor dx = empty({g.m, g.k}, x.dtype, dy.index), dw = empty({g.n, g.k}, dw_type, dy.index);
    at::Tensor dbias = empty({g.n}, at::kFloat, dy.index), work = empty({g.workspace_bytes}, at::kByte, dy.index);
    g.dy = dy.ptr; g.lddy = dy.ld; g.x = x.ptr; g.ldx = x.ld; g.wt = wt.ptr; g.ldwt = wt.ld;
    g.dx = dx.data_ptr(); g.lddx = g.k; g.dw = dw.data_ptr(); g.lddw = g.k;
    g.dbias = static_cast<float*>(dbias.data_ptr());
    g.workspace = work.data_ptr();
    const int rc = gemm_sm100a_int8_linear_backward(&g, stream_of(dy.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_int8_linear_backward", "");
    PyObject* const r = PyTuple_New(3);
    if (!r) throw Refused();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(dx)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(dw)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(dbias)));
    return r;
  });
}

// (x, transpose, dropout, column_sums) -> (q, scale) or (q, scale, sums)
PyObject* py_quantize(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 4);
    const Matrix x = matrix(v[0], "x", -1);
    const int code = floating(x, "x");
    const bool transpose = truth(v[1]), sums = truth(v[3]);
    if (sums && !transpose) refuse("column_sums needs transpose=True");
    if (!transpose && x.cols == 0 && x.rows > 0) refuse("x has no columns");
    Int8QuantArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.x_type = code;
    g.rows = x.rows; g.cols = x.cols;
    g.x = x.ptr; g.ldx = x.ld;
    g.transpose = transpose ? 1 : 0;
    g.drop = dropout_args(v[2], x.cols, x.index);
    at::Tensor q = transpose ? empty_int8(x.cols, x.rows, x.index) : empty_int8(x.rows, x.cols, x.index);
    at::Tensor scale = empty({transpose ? x.cols : x.rows}, at::kFloat, x.index), c;
    if (sums) {
      c = empty({x.cols}, at::kFloat, x.index);
      g.col_sums = static_cast<float*>(c.data_ptr());
    }
    g.q = q.data_ptr();
    g.ldq = q.stride(0);
    g.scale = static_cast<float*>(scale.data_ptr());
    if (scale.size(0) > 0) {
      const int rc = gemm_sm100a_quantize_int8(&g, stream_of(x.index));
      if (rc != GEMM_OK) failed(rc, "gemm_sm100a_quantize_int8", "");
    }
    PyObject* const r = PyTuple_New(sums ? 3 : 2);
    if (!r) throw Refused();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scale)));
    if (sums) PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(c)));
    return r;
  });
}

// (x, dropout, residual, out)
PyObject* py_dropout(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 4);
    const Matrix x = matrix(v[0], "x", -1);
    DropoutOpArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.type = floating(x, "x");
    g.rows = x.rows; g.cols = x.cols;
    g.x = x.ptr; g.ldx = x.ld;
    if (v[2] != Py_None) {
      const Matrix r = matrix(v[2], "residual", x.index);
      same_type(r, "residual", x.dtype);
      shape(r, "residual", x.rows, x.cols);
      g.residual = r.ptr;
      g.ldr = r.ld;
    }
    g.drop = dropout_args(v[1], x.cols, x.index);
    Output y = output(v[3], x.rows, x.cols, x.dtype, x.index);
    g.y = y.ptr;
    g.ldy = y.ld;
    const int rc = gemm_sm100a_dropout(&g, stream_of(x.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_dropout", "");
    return y.wrap();
  });
}

// ------------------------------------------------------------------ 4-bit operands
// An Fp4 tuple (values, scales, row_scale, cols, block).
struct Fp4Operand {
  void* values;
  int64_t rows, cols, ld;
  void* scales;
  const float* row_scale;
  int32_t block;
  int index;
};

const at::Tensor& bytes(PyObject* o, const char* name, const char* part, int dims, int index) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.dim() == dims && t.layout() == c10::kStrided && t.scalar_type() == at::kByte && t.is_cuda() && (index < 0 || t.get_device() == index))
      return t;
  }
  refuse("%s.%s must be a %d-D uint8 tensor on the operands' CUDA device", name, part, dims);
}

int32_t block_arg(PyObject* o) {
  const int64_t b = integer(o);
  if (b != 16 && b != 32) refuse("block must be 16 or 32");
  return (int32_t)b;
}

Fp4Operand fp4_operand(PyObject* o, const char* name, int index) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) refuse("%s must be an Fp4", name);
  Fp4Operand f;
  const at::Tensor& v = bytes(PyTuple_GET_ITEM(o, 0), name, "values", 2, index);
  f.index = v.get_device();
  const at::Tensor& s = bytes(PyTuple_GET_ITEM(o, 1), name, "scales", 1, f.index);
  f.cols = integer(PyTuple_GET_ITEM(o, 3));
  f.block = block_arg(PyTuple_GET_ITEM(o, 4));
  f.rows = v.size(0);
  if (f.cols < 0 || v.size(1) != (f.cols + 1) / 2)
    refuse("%s.values must have %lld columns for %lld elements", name, (long long)((f.cols + 1) / 2), (long long)f.cols);
  f.ld = v.stride(0);
  if (v.stride(1) != 1 && v.size(1) > 1) refuse("%s.values must have unit stride along its last axis", name);
  if (f.rows <= 1) f.ld = pad16(v.size(1));
  if ((f.ld & 15) || f.ld < v.size(1)) refuse("%s.values must have a row stride that is a multiple of 16 bytes", name);
  const int64_t need = gemm_sm100a_fp4_scale_bytes(f.rows, f.cols, f.block);
  if (need < 0) refuse("%s is too large", name);
  if (s.size(0) < need || (s.stride(0) != 1 && need > 1)) refuse("%s.scales must hold %lld contiguous bytes", name, (long long)need);
  f.values = v.data_ptr();
  f.scales = s.data_ptr();
  PyObject* const r = PyTuple_GET_ITEM(o, 2);
  f.row_scale = r == Py_None ? nullptr : static_cast<const float*>(vector(r, "row_scale", f.rows, f.index, nullptr));
  return f;
}

// (x, block) -> (values, scales, row_scale)
PyObject* py_quantize_fp4(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 2);
    const Matrix x = matrix(v[0], "x", -1);
    Fp4QuantArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.x_type = floating(x, "x");
    g.block = block_arg(v[1]);
    g.rows = x.rows; g.cols = x.cols;
    g.x = x.ptr; g.ldx = x.ld;
    if (x.cols == 0 && x.rows > 0) refuse("x has no columns");
    const int64_t scale_bytes = gemm_sm100a_fp4_scale_bytes(x.rows, x.cols, g.block);
    if (scale_bytes < 0) failed(GEMM_ERR_CANNOT_IMPLEMENT, "gemm_sm100a_quantize_fp4", "dimension too large");
    const int64_t width = (x.cols + 1) / 2;
    at::Tensor q = at::Tensor(at::detail::empty_strided_cuda({x.rows, width}, {row_bytes(width), 1}, at::kByte,
                                                             at::Device(at::kCUDA, (c10::DeviceIndex)x.index)));
    at::Tensor scales = empty({scale_bytes}, at::kByte, x.index), rows = empty({x.rows}, at::kFloat, x.index);
    g.values = q.data_ptr(); g.ldv = q.stride(0);
    g.scales = scales.data_ptr();
    g.row_scale = static_cast<float*>(rows.data_ptr());
    const int rc = gemm_sm100a_quantize_fp4(&g, stream_of(x.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_quantize_fp4", "");
    PyObject* const r = PyTuple_New(3);
    if (!r) throw Refused();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scales)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(rows)));
    return r;
  });
}

// (q, dtype, out)
PyObject* py_dequantize_fp4(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 3);
    const Fp4Operand q = fp4_operand(v[0], "q", -1);
    at::ScalarType t;
    if (v[2] != Py_None) {
      const Matrix d = matrix(v[2], "out", q.index);
      floating(d, "out");
      t = d.dtype;
    } else {
      t = dtype_arg(v[1], "dtype");
    }
    Output y = output(v[2], q.rows, q.cols, t, q.index);
    Fp4DequantArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.y_type = type_code(t);
    g.block = q.block;
    g.rows = q.rows; g.cols = q.cols;
    g.values = q.values; g.ldv = q.ld; g.scales = q.scales; g.row_scale = q.row_scale;
    g.y = y.ptr; g.ldy = y.ld;
    const int rc = gemm_sm100a_dequantize_fp4(&g, stream_of(q.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_dequantize_fp4", "");
    return y.wrap();
  });
}

// The part of Fp4GemmArgs that products and linear layers share.
void common_fp4(Fp4GemmArgs& g, PyObject* bias, PyObject* residual, PyObject* status, PyObject* const* knobs, at::ScalarType t, int index) {
  g.struct_size = sizeof(g);
  g.d_type = type_code(t);
  if (residual != Py_None) {
    const Matrix c = matrix(residual, "residual", index);
    same_type(c, "residual", t);
    shape(c, "residual", g.m, g.n);
    g.c = c.ptr;
    g.ldc = c.ld;
  }
  if (bias != Py_None) g.bias = vector(bias, "bias", g.n, index, &g.bias_type);
  g.status = status_word(status, index);
  g.tile_n = knob(knobs[0], "tile_n");
  g.cta_group = knob(knobs[1], "cta_group");
  g.split_k = knob(knobs[2], "split_k");
  g.timeout_ms = (uint32_t)knob(knobs[3], "timeout_ms");
  g.flags = (uint32_t)knob(knobs[4], "flags");
}

at::ScalarType result_type(PyObject* out, PyObject* dtype, const char* name, int index) {
  if (out == Py_None) return dtype_arg(dtype, name);
  const Matrix d = matrix(out, "out", index);
  floating(d, "out");
  return d.dtype;
}

[[noreturn]] void failed_fp4(int rc, const Fp4GemmArgs& g, const char* what) {
  GemmInfo info;
  gemm_sm100a_fp4_query(&g, &info);
  failed(rc, what, info.reason);
}

// (a, b, bias, residual, out_dtype, out, status, tile_n, cta_group, split_k, timeout_ms, flags)
PyObject* py_gemm_fp4(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 12);
    const Fp4Operand a = fp4_operand(v[0], "a", -1), b = fp4_operand(v[1], "b", a.index);
    if (b.cols != a.cols) refuse("b must have %lld columns, as a has, got %lld", (long long)a.cols, (long long)b.cols);
    if (b.block != a.block) refuse("b must have blocks of %d, as a has, got %d", (int)a.block, (int)b.block);
    Fp4GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.m = a.rows; g.n = b.rows; g.k = a.cols;
    g.block = a.block;
    const at::ScalarType t = result_type(v[5], v[4], "out_dtype", a.index);
    common_fp4(g, v[2], v[3], v[6], v + 7, t, a.index);
    Output d = output(v[5], g.m, g.n, t, a.index);
    g.a = a.values; g.lda = a.ld; g.a_scales = a.scales; g.a_row_scale = a.row_scale;
    g.b = b.values; g.ldb = b.ld; g.b_scales = b.scales; g.b_row_scale = b.row_scale;
    g.d = d.ptr; g.ldd = d.ld;
    const int rc = gemm_sm100a_fp4_launch(&g, stream_of(a.index));
    if (rc != GEMM_OK) failed_fp4(rc, g, "gemm_sm100a_fp4_launch");
    return d.wrap();
  });
}

// (x, w, bias, residual, out_dtype, out, status, tile_n, cta_group, split_k, timeout_ms, flags)
PyObject* py_linear_fp4(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 12);
    const Matrix x = matrix(v[0], "x", -1);
    const int code = floating(x, "x");
    const Fp4Operand w = fp4_operand(v[1], "w", x.index);
    if (w.cols != x.cols) refuse("w must have %lld columns, as x has, got %lld", (long long)x.cols, (long long)w.cols);
    Fp4GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.m = x.rows; g.n = w.rows; g.k = x.cols;
    g.block = w.block;
    const at::ScalarType t = v[5] == Py_None && v[4] == Py_None ? x.dtype : result_type(v[5], v[4], "out_dtype", x.index);
    common_fp4(g, v[2], v[3], v[6], v + 7, t, x.index);
    Output d = output(v[5], g.m, g.n, t, x.index);
    g.b = w.values; g.ldb = w.ld; g.b_scales = w.scales; g.b_row_scale = w.row_scale;
    g.d = d.ptr; g.ldd = d.ld;
    g.lda = row_bytes((g.k + 1) / 2);
    at::Tensor work;
    if (gemm_sm100a_fp4_linear_workspace(&g, x.ptr, code, x.ld)) {
      const int64_t values = g.m * g.lda, scales = gemm_sm100a_fp4_scale_bytes(g.m, g.k, g.block);
      if (scales < 0) failed(GEMM_ERR_CANNOT_IMPLEMENT, "gemm_sm100a_fp4_linear", "dimension too large");
      work = empty({values + scales + 4 * g.m + 16}, at::kByte, x.index);     // 4-bit tokens, their scales, their row scales
      uint8_t* const q = static_cast<uint8_t*>(work.data_ptr());
      g.a = q;
      g.a_scales = q + values;
      g.a_row_scale = reinterpret_cast<const float*>(q + values + scales);
    }
    const int rc = gemm_sm100a_fp4_linear(&g, x.ptr, code, x.ld, stream_of(x.index));
    if (rc != GEMM_OK) {
      if (!g.a) { g.a = g.b; g.a_scales = g.b_scales; }   // for the reason only
      failed_fp4(rc, g, "gemm_sm100a_fp4_linear");
    }
    return d.wrap();
  });
}

// ------------------------------------------------------------------ norms around a block
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused();
  return v;
}

// weight, post_weight and a vector gate: one type, x's or fp32.
struct Params {
  int32_t type;      // -1 before the first
  int32_t x_type;
  int64_t n;
  int index;
  const void* get(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    int32_t code;
    const void* p = vector(o, name, n, index, &code);
    if (code != x_type && code != GEMM_TYPE_FP32) refuse("%s must have x's type or be float32", name);
    if (type >= 0 && code != type) refuse("weight, post_weight and a gate vector must have one type");
    type = code;
    return p;
  }
};

// The gate: a vector of n elements (ld 0), or a matrix like x.
const void* gate_arg(PyObject* o, Params& params, const Matrix& x, int64_t& ld) {
  ld = 0;
  if (o == Py_None) return nullptr;
  if (THPVariable_Check(o) && THPVariable_Unpack(o).dim() == 2) {
    const Matrix g = matrix(o, "gate", x.index);
    same_type(g, "gate", x.dtype);
    shape(g, "gate", x.rows, x.cols);
    ld = g.ld;
    return g.ptr;
  }
  return params.get(o, "gate");
}

Matrix like(PyObject* o, const char* name, const Matrix& x) {
  const Matrix m = matrix(o, name, x.index);
  same_type(m, name, x.dtype);
  shape(m, name, x.rows, x.cols);
  return m;
}

// (x, y, weight, post_weight, gate, scale, eps, fp4, out) -> (x_out, h) or (x_out, values, scales, row_scale)
PyObject* py_residual_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 9);
    const Matrix x = matrix(v[0], "x", -1);
    ResidualNormArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.type = floating(x, "x");
    g.rows = x.rows; g.cols = x.cols;
    g.x = x.ptr; g.ldx = x.ld;
    Params params = {-1, g.type, x.cols, x.index};
    g.weight = params.get(v[2], "weight");
    const bool block = v[1] != Py_None;
    Output xo;
    if (block) {
      const Matrix y = like(v[1], "y", x);
      g.y = y.ptr; g.ldy = y.ld;
      g.post_weight = params.get(v[3], "post_weight");
      g.gate = gate_arg(v[4], params, x, g.ldg);
      xo = output(v[8], x.rows, x.cols, x.dtype, x.index);
      g.x_out = xo.ptr; g.ldo = xo.ld;
    } else {
      if (v[3] != Py_None || v[4] != Py_None || v[8] != Py_None) refuse("post_weight, gate and out need y");
      xo.given = v[0];
    }
    g.param_type = params.type < 0 ? g.type : params.type;
    g.scale = (float)real(v[5]);
    g.eps = real(v[6]);
    const int64_t four = integer(v[7]);
    if (four != 0 && four != 16 && four != 32) refuse("fp4 must be 0, 16 or 32");
    g.block = (int32_t)four;
    at::Tensor h, scales, rows;
    if (four) {
      const int64_t scale_bytes = gemm_sm100a_fp4_scale_bytes(x.rows, x.cols, g.block), width = (x.cols + 1) / 2;
      if (scale_bytes < 0) failed(GEMM_ERR_CANNOT_IMPLEMENT, "gemm_sm100a_residual_norm", "dimension too large");
      h = at::Tensor(at::detail::empty_strided_cuda({x.rows, width}, {row_bytes(width), 1}, at::kByte,
                                                    at::Device(at::kCUDA, (c10::DeviceIndex)x.index)));
      scales = empty({scale_bytes}, at::kByte, x.index);
      rows = empty({x.rows}, at::kFloat, x.index);
      g.values = h.data_ptr(); g.ldv = h.stride(0);
      g.scales = scales.data_ptr();
      g.row_scale = static_cast<float*>(rows.data_ptr());
    } else {
      h = empty({x.rows, x.cols}, x.dtype, x.index);
      g.h = h.data_ptr(); g.ldh = x.cols;
    }
    const int rc = gemm_sm100a_residual_norm(&g, stream_of(x.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_residual_norm", x.cols > 16384 || x.cols < 1 ? "1 to 16384 columns" : "");
    PyObject* const r = PyTuple_New(four ? 4 : 2);
    if (!r) throw Refused();
    PyTuple_SET_ITEM(r, 0, xo.wrap());
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(h)));
    if (four) {
      PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(scales)));
      PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(rows)));
    }
    return r;
  });
}

// (dh, dx_out, x_out, y, weight, post_weight, gate, scale, eps) -> (dx, dy, dweight, dpost_weight, dgate)
PyObject* py_residual_norm_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 9);
    const Matrix x = matrix(v[2], "x_out", -1);
    ResidualNormBackwardArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.type = floating(x, "x_out");
    g.rows = x.rows; g.cols = x.cols;
    g.x_out = x.ptr; g.ldo = x.ld;
    const Matrix dh = like(v[0], "dh", x);
    g.dh = dh.ptr; g.lddh = dh.ld;
    if (v[1] != Py_None) {
      const Matrix d = like(v[1], "dx_out", x);
      g.dx_out = d.ptr; g.lddo = d.ld;
    }
    Params params = {-1, g.type, x.cols, x.index};
    g.weight = params.get(v[4], "weight");
    const bool block = v[3] != Py_None;
    if (block) {
      const Matrix y = like(v[3], "y", x);
      g.y = y.ptr; g.ldy = y.ld;
      g.post_weight = params.get(v[5], "post_weight");
      g.gate = gate_arg(v[6], params, x, g.ldg);
    } else if (v[5] != Py_None || v[6] != Py_None) {
      refuse("post_weight and gate need y");
    }
    g.param_type = params.type < 0 ? g.type : params.type;
    g.scale = (float)real(v[7]);
    g.eps = real(v[8]);
    g.workspace_bytes = gemm_sm100a_residual_norm_workspace(x.rows, x.cols);
    if (g.workspace_bytes < 0) failed(GEMM_ERR_CANNOT_IMPLEMENT, "gemm_sm100a_residual_norm_backward", "1 to 16384 columns");
    const at::Tensor dx = empty({x.rows, x.cols}, x.dtype, x.index), work = empty({g.workspace_bytes}, at::kByte, x.index);
    at::Tensor dy, dw, dp, dg;
    g.dx = dx.data_ptr(); g.lddx = x.cols;
    g.workspace = work.data_ptr();
    if (block) {
      dy = empty({x.rows, x.cols}, x.dtype, x.index);
      g.dy = dy.data_ptr(); g.lddy = x.cols;
    }
    if (g.weight) {
      dw = empty({x.cols}, at::kFloat, x.index);
      g.dweight = static_cast<float*>(dw.data_ptr());
    }
    if (g.post_weight) {
      dp = empty({x.cols}, at::kFloat, x.index);
      g.dpost_weight = static_cast<float*>(dp.data_ptr());
    }
    if (g.gate) {
      dg = g.ldg ? empty({x.rows, x.cols}, x.dtype, x.index) : empty({x.cols}, at::kFloat, x.index);
      g.dgate = dg.data_ptr(); g.lddg = x.cols;
    }
    const int rc = gemm_sm100a_residual_norm_backward(&g, stream_of(x.index));
    if (rc != GEMM_OK) failed(rc, "gemm_sm100a_residual_norm_backward", "");
    PyObject* const r = PyTuple_New(5);
    if (!r) throw Refused();
    const at::Tensor* const all[5] = {&dx, &dy, &dw, &dp, &dg};
    for (int i = 0; i < 5; ++i) {
      if (all[i]->defined()) {
        PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*all[i]));
      } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(r, i, Py_None);
      }
    }
    return r;
  });
}

// (rows, cols, device index)
PyObject* py_empty(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&] {
    count(n, 3);
    return THPVariable_Wrap(empty_int8(integer(v[0]), integer(v[1]), (int)integer(v[2])));
  });
}

PyObject* py_set_raise(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XDECREF(g_raise);
  g_raise = f;
  Py_RETURN_NONE;
}

#define FAST(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    FAST("gemm", py_gemm), FAST("linear", py_linear), FAST("backward", py_backward), FAST("quantize", py_quantize),
    FAST("dropout", py_dropout), FAST("empty", py_empty),
    FAST("quantize_fp4", py_quantize_fp4), FAST("dequantize_fp4", py_dequantize_fp4), FAST("gemm_fp4", py_gemm_fp4),
    FAST("linear_fp4", py_linear_fp4), FAST("residual_norm", py_residual_norm),
    FAST("residual_norm_backward", py_residual_norm_backward), {"set_raise", py_set_raise, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "gemm_sm100a_torch", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit_gemm_sm100a_torch(void) { return PyModule_Create(&g_module); }
