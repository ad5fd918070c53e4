// dropout.cu -- Y = residual + dropout(X) with a mask that is never stored: it
// is drawn again from the counter of each element (counter_rng.cuh) wherever it
// is needed.  Bound by the bytes of X, residual and Y.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "gemm_sm100a.h"
#include "int8_common.cuh"
#include "sm100_ptx.cuh"

using namespace int8op;

namespace {

struct DropoutParams {
  const void* x; int64_t ldx;
  const void* res; int64_t ldr;
  void* y; int64_t ldy;
  int64_t rows, cols;
  Drop drop;
  int32_t wide;
};

// One 16-byte vector per thread and row; blockDim.x threads cover a segment of
// the row, blockDim.y rows.  A thread walks down its column of vectors,
// so the key, the pointers and the addresses cost little per vector:
// drawing the mask (two 64-bit products per pair of elements) is what bounds the
// kernel next to the bytes.
template <typename T, bool RES, bool ON>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int V = Vec<T>::N;
  constexpr int UN = sizeof(T) == 4 ? 2 : 1;   // rows at a time (16384 x 8192 bf16 with residual 127 us, 133 with two)
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  if (c >= p.cols) return;
  const int n = (int)min((int64_t)V, p.cols - c);
  const uint64_t key = ON ? drop_key(p.drop) : 0;
  const F2 grow2(ON ? p.drop.grow : 1.f, ON ? p.drop.grow : 1.f);
  const uint32_t threshold = p.drop.threshold;
  const int64_t step = (int64_t)gridDim.y * blockDim.y;
  for (int64_t r0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r0 < p.rows; r0 += UN * step) {
    Vec<T> v[UN], b[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t r = r0 + u * step;
      const int nn = r < p.rows ? n : 0;
      v[u] = load_vec<T>(static_cast<const T*>(p.x) + r * p.ldx + c, nn, p.wide);
      if constexpr (RES) b[u] = load_vec<T>(static_cast<const T*>(p.res) + r * p.ldr + c, nn, p.wide);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t r = r0 + u * step;
      if (r >= p.rows) break;
      uint32_t w[V];
      if constexpr (ON) drop_words<V>(p.drop, key, drop_index(p.drop, r, c), w);
      Vec<T> o;
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        F2 x(!ON || w[j] >= threshold ? v[u].get(j) : 0.f, !ON || w[j + 1] >= threshold ? v[u].get(j + 1) : 0.f);
        x = RES ? fma2(x, grow2, F2(b[u].get(j), b[u].get(j + 1))) : mul2(x, grow2);
        float f0, f1;
        x.get(f0, f1);
        o.set2(j, f0, f1);
      }
      store_vec<T>(static_cast<T*>(p.y) + r * p.ldy + c, o, n, p.wide);
    }
  }
}

template <typename T>
cudaError_t launch(const DropoutParams& p, cudaStream_t st) {
  const int64_t nvec = (p.cols + Vec<T>::N - 1) / Vec<T>::N;
  int tx = 32;
  while (tx < 256 && tx < nvec) tx *= 2;
  const int ty = 256 / tx;
  const int64_t gx = (nvec + tx - 1) / tx;
  int64_t gy = (p.rows + ty - 1) / ty;
  const int64_t most = (148 * 16 + gx - 1) / gx;      // two waves of blocks and more rows per thread
  if (gy > most) gy = most;
  const dim3 grid((unsigned)gx, (unsigned)gy), block((unsigned)tx, (unsigned)ty);
  void (*fn)(DropoutParams) = p.drop.on ? (p.res ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                                        : (p.res ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
  return launch_overlapped(fn, grid, block, 0, 1, st, p);
}

}  // namespace

extern "C" int gemm_sm100a_dropout(const DropoutOpArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(DropoutOpArgs)) return GEMM_ERR_BAD_ARGS;
  if (!type_ok(a->type) || a->rows < 0 || a->cols < 0 || a->cols > INT32_MAX / 2 || a->rows > INT32_MAX / 2)
    return GEMM_ERR_CANNOT_IMPLEMENT;
  DropoutParams p;
  memset(&p, 0, sizeof(p));
  const char* why = "";
  const int rc = drop_resolve(a->drop, a->rows, a->cols, p.drop, &why);
  if (rc != GEMM_OK) return rc;
  if (a->rows == 0 || a->cols == 0) return GEMM_OK;
  if (!a->x || !a->y) return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->type);
  if (a->ldx < a->cols || a->ldy < a->cols || (a->residual && a->ldr < a->cols)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if ((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->y) | reinterpret_cast<uintptr_t>(a->residual)) % e)
    return GEMM_ERR_CANNOT_IMPLEMENT;
  // A shifted overlap would read elements that other threads have stored already.
  if (!in_place_or_apart(a->x, a->ldx, a->y, a->ldy, a->rows, a->cols, e) ||
      (a->residual && !in_place_or_apart(a->residual, a->ldr, a->y, a->ldy, a->rows, a->cols, e)))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  p.x = a->x; p.ldx = a->ldx; p.res = a->residual; p.ldr = a->ldr; p.y = a->y; p.ldy = a->ldy;
  p.rows = a->rows; p.cols = a->cols;
  p.wide = rows_16b(a->x, a->ldx, e) && rows_16b(a->y, a->ldy, e) && (!a->residual || rows_16b(a->residual, a->ldr, e));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->y);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const cudaError_t err = a->type == GEMM_TYPE_BF16 ? launch<__nv_bfloat16>(p, st)
                        : a->type == GEMM_TYPE_FP16 ? launch<__half>(p, st) : launch<float>(p, st);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}
