// int8_backward.cu -- the gradients of the int8 linear layer in one call: three
// quantisations of dY and X and two products, all of them the library's own kernels.
//
//   dZ = dropout(dY),  dX = dZ . W,  dW = dZ^T . X,  dbias = column sums of dZ
//
// dX contracts over the channels and dW over the tokens, so dZ is quantised twice: along
// its rows and, transposed, along its columns (which also gives dbias); X along its columns.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "gemm_sm100a.h"
#include "int8_common.cuh"

using namespace int8op;

namespace {

constexpr int64_t kMaxK = 131071;

// Rows of whole 128-byte lines: a TMA row of an operand then never straddles two.
int64_t row_bytes(int64_t cols) { return (cols + 127) / 128 * 128; }

struct Workspace {
  int64_t z, zt, xt, z_scale, zt_scale, xt_scale, total;   // byte offsets
};

Workspace layout(int64_t m, int64_t n, int64_t k) {
  Workspace w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t here = at; at += (bytes + 127) / 128 * 128; return here; };
  w.z = take(m * row_bytes(n));
  w.zt = take(n * row_bytes(m));
  w.xt = take(k * row_bytes(m));
  w.z_scale = take(m * 4);
  w.zt_scale = take(n * 4);
  w.xt_scale = take(k * 4);
  w.total = at;
  return w;
}

}  // namespace

extern "C" int64_t gemm_sm100a_int8_backward_workspace(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0 || m > kMaxK || n > kMaxK || k > INT32_MAX / 2) return -1;
  return layout(m, n, k).total;
}

extern "C" int gemm_sm100a_int8_linear_backward(const Int8BackwardArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(Int8BackwardArgs)) return GEMM_ERR_BAD_ARGS;
  const int64_t m = a->m, n = a->n, k = a->k;
  if (!type_ok(a->type) || !type_ok(a->dw_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (m < 0 || n <= 0 || k <= 0 || m > kMaxK || n > kMaxK || k > INT32_MAX / 2) return GEMM_ERR_CANNOT_IMPLEMENT;
  // Everything the calls below would refuse is refused here, before the first launch.
  const uintptr_t e = (uintptr_t)type_bytes(a->type), ew = (uintptr_t)type_bytes(a->dw_type);
  auto off = [](const void* p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by != 0; };
  Drop drop;
  const char* why = "";
  if (drop_resolve(a->drop, m, n, drop, &why) != GEMM_OK) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!a->dx && !a->dw && !a->dbias) return GEMM_OK;
  if (off(a->dx, e) || off(a->dw, ew) || off(a->dbias, 4) || (a->dx && a->lddx < k) || (a->dw && a->lddw < k))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (m > 0) {
    if (!a->dy || (a->dw && !a->x) || (a->dx && (!a->wt || !a->wt_scale)) || !a->workspace) return GEMM_ERR_BAD_ARGS;
    if (off(a->dy, e) || a->lddy < n || off(a->workspace, 16)) return GEMM_ERR_CANNOT_IMPLEMENT;
    if (a->dw && (off(a->x, e) || a->ldx < k)) return GEMM_ERR_CANNOT_IMPLEMENT;
    if (a->dx && (off(a->wt, 16) || a->ldwt < n || a->ldwt % 16 != 0 || off(a->wt_scale, 4))) return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  const Workspace w = layout(m, n, k);
  if (m > 0 && a->workspace_bytes < w.total) return GEMM_ERR_BAD_ARGS;
  PointerDeviceGuard guard(a->dx ? a->dx : (a->dw ? a->dw : a->dbias));
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (m == 0) {
    if ((a->dw && cudaMemset2DAsync(a->dw, (size_t)a->lddw * ew, 0, (size_t)k * ew, (size_t)n, st) != cudaSuccess) ||
        (a->dbias && cudaMemsetAsync(a->dbias, 0, (size_t)n * 4, st) != cudaSuccess)) {
      cudaGetLastError();
      return GEMM_ERR_LAUNCH;
    }
    return GEMM_OK;
  }
  uint8_t* const ws = static_cast<uint8_t*>(a->workspace);
  auto quantize = [&](const void* x, int64_t cols, int64_t ld, bool transpose, const DropoutArgs* dr, int64_t q, int64_t scale,
                      float* sums) {
    Int8QuantArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.x_type = a->type; g.rows = m; g.cols = cols; g.x = x; g.ldx = ld;
    g.q = ws + q; g.ldq = row_bytes(transpose ? m : cols); g.scale = reinterpret_cast<float*>(ws + scale);
    g.transpose = transpose ? 1 : 0; g.col_sums = sums;
    if (dr) g.drop = *dr;
    return gemm_sm100a_quantize_int8(&g, stream);
  };
  auto product = [&](int64_t rows, int64_t cols, int64_t depth, const void* qa, int64_t lda, const float* sa, const void* qb,
                     int64_t ldb, const float* sb, void* d, int64_t ldd, int32_t type) {
    Int8GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.struct_size = sizeof(g);
    g.d_type = type; g.m = rows; g.n = cols; g.k = depth;
    g.a = qa; g.lda = lda; g.scale_a = sa; g.b = qb; g.ldb = ldb; g.scale_b = sb; g.d = d; g.ldd = ldd;
    g.status = a->status;
    return gemm_sm100a_int8_launch(&g, stream);
  };
  const float* const zs = reinterpret_cast<const float*>(ws + w.z_scale);
  const float* const zts = reinterpret_cast<const float*>(ws + w.zt_scale);
  const float* const xts = reinterpret_cast<const float*>(ws + w.xt_scale);
  int rc = GEMM_OK;
  // All quantisations before the first product: dX and dW may replace X or dY.
  if (a->dx) rc = quantize(a->dy, n, a->lddy, false, &a->drop, w.z, w.z_scale, nullptr);
  if (rc == GEMM_OK && (a->dw || a->dbias)) rc = quantize(a->dy, n, a->lddy, true, &a->drop, w.zt, w.zt_scale, a->dbias);
  if (rc == GEMM_OK && a->dw) rc = quantize(a->x, k, a->ldx, true, nullptr, w.xt, w.xt_scale, nullptr);
  if (rc == GEMM_OK && a->dx)
    rc = product(m, k, n, ws + w.z, row_bytes(n), zs, a->wt, a->ldwt, a->wt_scale, a->dx, a->lddx, a->type);
  if (rc == GEMM_OK && a->dw)
    rc = product(n, k, m, ws + w.zt, row_bytes(m), zts, ws + w.xt, row_bytes(m), xts, a->dw, a->lddw, a->dw_type);
  return rc;
}
