// int8_quantize.cu -- symmetric int8 quantisation with one scale per row, or
// per column with a transposed result (the operands of gemm_sm100a_int8_launch).
//
//   amax = max |x| over the row (column),  q = rint(127 x / amax),  scale = amax / 127
//
// Both kernels read X once from HBM and write one byte per element; they are
// bound by those bytes.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "gemm_sm100a.h"
#include "int8_common.cuh"
#include "sm100_ptx.cuh"

namespace cg = cooperative_groups;
using namespace int8op;

namespace {

struct QuantParams {
  const void* x;
  int64_t ldx, rows, cols;
  uint8_t* q;
  int64_t ldq;
  float* scale;
  float* col_sums;
  Drop drop;
  int32_t wide;         // every row of X starts on a 16-byte boundary
  int32_t row_chunk;    // columns kernel: rows of one CTA of the cluster
  int32_t rows_held;    // columns kernel: how many of them stay in shared memory
};

// ----------------------------------------------------------------- rows
// A row belongs to blockDim.x threads (a block holds blockDim.y rows); each
// keeps NV 16-byte vectors in registers between the maximum and the rounding,
// so X is read once.  Rows longer than NV * blockDim.x vectors are read again
// (from L2) chunk by chunk.
template <typename T, int NV, bool DROP>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const __grid_constant__ QuantParams p) {
  constexpr int V = Vec<T>::N;
  __shared__ uint32_t warp_max[32];
  const int tx = threadIdx.x, TX = blockDim.x;
  const int nvec = (int)((p.cols + V - 1) / V);
  const int per_chunk = NV * TX;
  const int chunks = (nvec + per_chunk - 1) / per_chunk;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const uint64_t key = DROP ? drop_key(p.drop) : 0;
  for (int64_t row0 = (int64_t)blockIdx.x * blockDim.y; row0 < p.rows; row0 += (int64_t)gridDim.x * blockDim.y) {
    const int64_t row = row0 + threadIdx.y;
    const bool live = row < p.rows;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    Vec<T> v[NV];
    auto load = [&](int chunk) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (chunk * per_chunk + i * TX + tx) * V;
        v[i] = load_vec<T>(x + e, live ? (int)min((int64_t)V, p.cols - e) : 0, p.wide);
      }
      if constexpr (DROP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int64_t e = (int64_t)(chunk * per_chunk + i * TX + tx) * V;
          const uint32_t keep = drop_mask<V>(key, p.drop.threshold, drop_index(p.drop, row, e));
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!(keep >> j & 1u)) v[i].zero(j);
        }
      }
    };
    uint32_t top = 0;   // largest |x| so far: packed halves (16-bit T) or fp32 bits
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) top = max(top, v[i].w[j] & 0x7FFFFFFFu);
          else top = __vmaxu2(top, v[i].w[j] & 0x7FFF7FFFu);
        }
    }
    if constexpr (sizeof(T) == 2) top = abs_bits_to_f32<T>(max(top & 0xFFFFu, top >> 16));
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (TX > 32) {
      const int warp = threadIdx.y * (TX >> 5) + (tx >> 5);
      if ((tx & 31) == 0) warp_max[warp] = top;
      __syncthreads();
      const int w = tx & 31;
      top = __reduce_max_sync(0xFFFFFFFFu, w < (TX >> 5) ? warp_max[threadIdx.y * (TX >> 5) + w] : 0u);
      __syncthreads();
    }
    const RowScale s = row_scale(top);
    if (live && tx == 0) p.scale[row] = DROP ? s.scale * p.drop.grow : s.scale;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (c * per_chunk + i * TX + tx) * V;
        if (!live || e >= p.cols) continue;
        uint32_t w[V / 4];
        quantize_vec<T>(v[i], s, w);
        uint8_t* q = p.q + row * p.ldq + e;
        if (p.cols - e >= V) {
          if constexpr (V == 8) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
          else *reinterpret_cast<uint32_t*>(q) = w[0];
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (e + j < p.cols) q[j] = (uint8_t)(w[j / 4] >> (8 * (j & 3)));
        }
      }
    }
  }
}

// ----------------------------------------------------------------- columns
// A cluster owns a strip of 64 columns; its CTAs split the rows.  Each CTA
// reads its rows once, keeps them in shared memory and finds the column
// maxima (and sums); the cluster combines them through distributed shared
// memory; then every thread rounds 32 rows of two columns and writes two
// whole 32-byte sectors of the transposed result.
constexpr int kStrip = 64;
constexpr int kColThreads = 256;

template <typename T, bool DROP>
__global__ void __launch_bounds__(kColThreads) quantize_cols_kernel(const __grid_constant__ QuantParams p) {
  constexpr int V = Vec<T>::N;
  constexpr int LANES = kStrip / V;            // threads that cover one row of the strip
  constexpr int RPP = kColThreads / LANES;     // rows read per pass
  extern __shared__ __align__(16) uint8_t smem[];
  T* const held = reinterpret_cast<T*>(smem);  // [rows_held][kStrip]
  __shared__ uint32_t part_max[RPP][kStrip];
  __shared__ float part_sum[RPP][kStrip];
  __shared__ uint32_t cta_max[kStrip];
  __shared__ float cta_sum[kStrip];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), peers = (int)cluster.num_blocks();
  const int64_t col0 = (int64_t)(blockIdx.x / peers) * kStrip;
  const int64_t row0 = (int64_t)rank * p.row_chunk;
  const int n_rows = (int)max((int64_t)0, min((int64_t)p.row_chunk, p.rows - row0));
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const uint64_t key = DROP ? drop_key(p.drop) : 0;

  const int lane_c = threadIdx.x % LANES, lane_r = threadIdx.x / LANES;
  const int64_t c = col0 + lane_c * V;
  const int n_valid = (int)max((int64_t)0, min((int64_t)V, p.cols - c));
  const T* const x = static_cast<const T*>(p.x);
  uint32_t top[V];
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) { top[j] = 0u; sum[j] = 0.f; }
  constexpr int UN = 4;   // rows in flight per thread
  for (int r = lane_r; r < n_rows; r += UN * RPP) {
    Vec<T> v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int rr = r + u * RPP;
      v[u] = load_vec<T>(x + (row0 + rr) * p.ldx + c, rr < n_rows ? n_valid : 0, p.wide);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int rr = r + u * RPP;
      if (rr >= n_rows) break;
      if constexpr (DROP) {
        const uint32_t keep = drop_mask<V>(key, p.drop.threshold, drop_index(p.drop, row0 + rr, c));
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!(keep >> j & 1u)) v[u].zero(j);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float f = v[u].get(j);
        top[j] = max(top[j], __float_as_uint(f) & 0x7FFFFFFFu);
        sum[j] += f;
      }
      if (rr < p.rows_held)
        *reinterpret_cast<uint4*>(held + rr * kStrip + lane_c * V) = make_uint4(v[u].w[0], v[u].w[1], v[u].w[2], v[u].w[3]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    part_max[lane_r][lane_c * V + j] = top[j];
    part_sum[lane_r][lane_c * V + j] = sum[j];
  }
  __syncthreads();
  if (threadIdx.x < kStrip) {
    uint32_t m = 0;
    float s = 0.f;
    for (int r = 0; r < RPP; ++r) {
      m = max(m, part_max[r][threadIdx.x]);
      s += part_sum[r][threadIdx.x];
    }
    cta_max[threadIdx.x] = m;
    cta_sum[threadIdx.x] = s;
  }
  cluster.sync();
  // Every thread of warp w works on columns 2 * lane and 2 * lane + 1.
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t m0 = 0, m1 = 0;
  float s0 = 0.f, s1 = 0.f;
  for (int i = 0; i < peers; ++i) {
    const uint32_t* pm = cluster.map_shared_rank(cta_max, i);
    m0 = max(m0, pm[2 * lane]);
    m1 = max(m1, pm[2 * lane + 1]);
    if (rank == 0 && warp == 0 && p.col_sums) {
      const float* ps = cluster.map_shared_rank(cta_sum, i);
      s0 += ps[2 * lane];
      s1 += ps[2 * lane + 1];
    }
  }
  const RowScale q0 = row_scale(m0), q1 = row_scale(m1);
  const int64_t c0 = col0 + 2 * lane;
  if (rank == 0 && warp == 0) {
    const float grow = DROP ? p.drop.grow : 1.f;
    if (c0 < p.cols) { p.scale[c0] = q0.scale * grow; if (p.col_sums) p.col_sums[c0] = s0 * grow; }
    if (c0 + 1 < p.cols) { p.scale[c0 + 1] = q1.scale * grow; if (p.col_sums) p.col_sums[c0 + 1] = s1 * grow; }
  }
  auto value = [&](int r, int64_t col) -> float {   // a row that did not fit: read and masked again
    if (col >= p.cols) return 0.f;
    if (DROP && !drop_keeps(key, p.drop.threshold, drop_index(p.drop, row0 + r, col))) return 0.f;
    return to_f32(x[(row0 + r) * p.ldx + col]);
  };
  for (int g = warp * 32; g < n_rows; g += (kColThreads / 32) * 32) {
    uint32_t w0[8], w1[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t b0[4], b1[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = g + 4 * k + j;
        float f0 = 0.f, f1 = 0.f;
        if (r < n_rows) {
          if (r < p.rows_held) {
            f0 = to_f32(held[r * kStrip + 2 * lane]);
            f1 = to_f32(held[r * kStrip + 2 * lane + 1]);
          } else {
            f0 = value(r, c0);
            f1 = value(r, c0 + 1);
          }
        }
        b0[j] = quantize_one<T>(f0, q0);
        b1[j] = quantize_one<T>(f1, q1);
      }
      w0[k] = q0.c == 0.f ? 0u : pack4(b0[0], b0[1], b0[2], b0[3]);
      w1[k] = q1.c == 0.f ? 0u : pack4(b1[0], b1[1], b1[2], b1[3]);
    }
    auto store = [&](int64_t col, const uint32_t (&w)[8]) {
      if (col >= p.cols) return;
      uint8_t* q = p.q + col * p.ldq + row0 + g;
      if (n_rows - g >= 32) {
        reinterpret_cast<uint4*>(q)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(q)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (g + j < n_rows) q[j] = (uint8_t)(w[j / 4] >> (8 * (j & 3)));
      }
    };
    store(c0, w0);
    store(c0 + 1, w1);
  }
  cluster.sync();   // peers may still read this CTA's maxima
}

// ----------------------------------------------------------------- host
template <typename T>
cudaError_t launch_rows(const QuantParams& p, cudaStream_t st) {
  constexpr int NV = 4;
  const int64_t nvec = (p.cols + Vec<T>::N - 1) / Vec<T>::N;
  int64_t tx = (nvec + NV - 1) / NV;
  tx = (tx + 31) / 32 * 32;
  if (tx > 1024) tx = 1024;
  const int ry = tx >= 256 ? 1 : (int)(256 / tx);
  int64_t blocks = (p.rows + ry - 1) / ry;
  if (blocks > 0x7FFFFFFF) blocks = 0x7FFFFFFF;
  const dim3 block((unsigned)tx, (unsigned)ry);
  return launch_overlapped(p.drop.on ? quantize_rows_kernel<T, NV, true> : quantize_rows_kernel<T, NV, false>,
                           dim3((unsigned)blocks), block, 0, 1, st, p);
}

template <typename T>
cudaError_t launch_cols(QuantParams p, cudaStream_t st) {
  constexpr int64_t kHeldBytes = 192 * 1024;
  int peers = (int)((p.rows + 255) / 256);
  peers = peers < 1 ? 1 : (peers > 8 ? 8 : peers);
  p.row_chunk = (int32_t)(((p.rows + peers - 1) / peers + 31) / 32 * 32);
  const int64_t fit = kHeldBytes / (kStrip * (int64_t)sizeof(T));
  p.rows_held = (int32_t)(p.row_chunk < fit ? p.row_chunk : fit);
  const int64_t strips = (p.cols + kStrip - 1) / kStrip;
  auto fn = p.drop.on ? quantize_cols_kernel<T, true> : quantize_cols_kernel<T, false>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kHeldBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(fn, dim3((unsigned)(strips * peers)), dim3(kColThreads),
                           (size_t)(p.rows_held * (int64_t)(kStrip * sizeof(T))), peers, st, p);
}

}  // namespace

extern "C" int gemm_sm100a_quantize_int8(const Int8QuantArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(Int8QuantArgs)) return GEMM_ERR_BAD_ARGS;
  if (!type_ok(a->x_type) || a->rows < 0 || a->cols < 0 || a->rows > INT32_MAX / 2 || a->cols > INT32_MAX / 2)
    return GEMM_ERR_CANNOT_IMPLEMENT;
  const bool tr = a->transpose != 0;
  const int64_t out_rows = tr ? a->cols : a->rows, out_cols = tr ? a->rows : a->cols;
  if (out_rows == 0 || (!tr && out_cols == 0)) return GEMM_OK;
  if (!a->scale || (a->rows > 0 && (!a->x || !a->q)) || (a->col_sums && !tr)) return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->x_type);
  if (a->rows > 0 && (a->ldx < a->cols || (reinterpret_cast<uintptr_t>(a->x) % e) != 0 || a->ldq < out_cols ||
                      a->ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(a->q) & 15) != 0))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if ((reinterpret_cast<uintptr_t>(a->scale) | reinterpret_cast<uintptr_t>(a->col_sums)) & 3) return GEMM_ERR_CANNOT_IMPLEMENT;
  QuantParams p;
  memset(&p, 0, sizeof(p));
  const char* why = "";
  const int rc = drop_resolve(a->drop, a->rows, a->cols, p.drop, &why);
  if (rc != GEMM_OK) return rc;
  p.x = a->x; p.ldx = a->ldx; p.rows = a->rows; p.cols = a->cols;
  p.q = static_cast<uint8_t*>(a->q); p.ldq = a->ldq; p.scale = a->scale; p.col_sums = a->col_sums;
  p.wide = rows_16b(a->x, a->ldx, e) ? 1 : 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->scale);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  cudaError_t err;
  switch (a->x_type * 2 + (tr ? 1 : 0)) {
    case 0: err = launch_rows<__nv_bfloat16>(p, st); break;
    case 1: err = launch_cols<__nv_bfloat16>(p, st); break;
    case 2: err = launch_rows<__half>(p, st); break;
    case 3: err = launch_cols<__half>(p, st); break;
    case 4: err = launch_rows<float>(p, st); break;
    default: err = launch_cols<float>(p, st); break;
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}
