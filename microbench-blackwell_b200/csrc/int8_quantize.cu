// int8_quantize.cu -- symmetric int8 quantisation with one scale per row, or
// per column with a transposed result (the operands of gemm_sm100a_int8_launch).
//
//   amax = max |x| over the row (column),  q = rint(127 x / amax),  scale = amax / 127
//
// Both kernels read X once from HBM and write one byte per element.  Rows longer than a
// block's registers, and columns longer than the shared memory of a cluster, are read
// a second time, from L2.
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
  int32_t rows_held;    // columns kernel: how many of them are in shared memory at a time (a multiple of 16)
};

// ----------------------------------------------------------------- rows
// Most threads of a row that keep nv vectors each (32768 16-bit values in all; 16384 for nv = 2).
__host__ __device__ constexpr int row_threads(int nv) { return nv < 4 ? 1024 : 4096 / nv; }

// A row belongs to blockDim.x threads (a block holds blockDim.y rows); each
// keeps NV 16-byte vectors in registers between the maximum and the rounding,
// so X is read once.  Rows longer than NV * blockDim.x vectors are read again
// (from L2) chunk by chunk.
template <typename T, int NV, bool DROP>
__global__ void __launch_bounds__(row_threads(NV)) quantize_rows_kernel(const __grid_constant__ QuantParams p) {
  constexpr int V = Vec<T>::N;
  __shared__ uint32_t warp_max[32];
  const int tx = threadIdx.x, TX = blockDim.x;
  const int nvec = (int)((p.cols + V - 1) / V);
  const int per_chunk = NV * TX;
  const int chunks = (nvec + per_chunk - 1) / per_chunk;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const uint64_t key = DROP ? drop_key(p.drop) : 0;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
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
        drop_vec<T>(p.drop, key, drop_index(p.drop, row, e), v[i]);
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

// ----------------------------------------------------------------- columns
// A cluster owns a strip of columns, 64 bytes of each row; its CTAs split the
// rows.  Each CTA copies its rows to shared memory with every load in flight at
// once, finds the column maxima (and sums) there, combines them with its peers
// through distributed shared memory, and rounds 16 rows of two columns per
// thread into 16-byte stores (whole 32-byte sectors per column) of the transposed
// result.  A strip of 512 or 1024 rows at a time leaves room for several CTAs per SM,
// whose phases overlap; the rows before the last such batch are read a second time,
// from L2 (the strips at work at one time are smaller than it).
constexpr int kStripBytes = 64;
// Rows of a CTA in shared memory at a time: with fewer, more CTAs overlap their
// phases, but more rows are read (and masked) twice.  8192 x 28672 bf16: 170 us
// with 512, 206 with 1024; with dropout and sums 397 and 330 (kernel times, from a graph).
constexpr int rows_held(bool drop) { return drop ? 1024 : 512; }

// Byte of row r in the held strip: a 64-byte gap after every 16 rows puts rows 16
// apart, which the lanes of a warp read together, in different banks.
__device__ __forceinline__ int held_at(int r) { return (r + (r >> 4)) * kStripBytes; }

template <typename T, bool DROP, int kColWarps>
__global__ void __launch_bounds__(32 * kColWarps) quantize_cols_kernel(const __grid_constant__ QuantParams p) {
  constexpr int kColThreads = 32 * kColWarps;
  constexpr int V = Vec<T>::N;
  constexpr int COLS = kStripBytes / (int)sizeof(T);
  constexpr int LANES = kStripBytes / 16;      // threads that cover one row of the strip
  constexpr int RPP = kColThreads / LANES;     // rows per pass of the block
  constexpr int PAIRS = COLS / 2;              // lanes that cover the strip two columns each
  constexpr int SETS = 32 / PAIRS;             // 16-row sets a warp rounds at once
  extern __shared__ __align__(16) uint8_t held[];
  __shared__ uint32_t part_max[kColWarps][COLS];
  __shared__ float part_sum[kColWarps][COLS];
  __shared__ uint32_t cta_max[COLS];
  __shared__ float cta_sum[COLS];
  __shared__ RowScale scales[COLS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), peers = (int)cluster.num_blocks();
  const int64_t col0 = (int64_t)(blockIdx.x / peers) * COLS;
  const int64_t row0 = (int64_t)rank * p.row_chunk;
  const int n_rows = (int)max((int64_t)0, min((int64_t)p.row_chunk, p.rows - row0));
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const uint64_t key = DROP ? drop_key(p.drop) : 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lane_c = threadIdx.x % LANES, lane_r = threadIdx.x / LANES;
  const int64_t c = col0 + lane_c * V;
  const int n_valid = (int)max((int64_t)0, min((int64_t)V, p.cols - c));
  const T* const x = static_cast<const T*>(p.x) + row0 * p.ldx;
  const uint32_t held_s = sm100::smem_u32(held);
  const uint32_t own_s = held_s + (uint32_t)(held_at(lane_r) + lane_c * 16);   // this thread's first 16 bytes
  constexpr uint32_t kPass = (RPP + RPP / 16) * kStripBytes;                     // and RPP rows on
  const int64_t pass_elems = RPP * p.ldx;
  // Rows [b * rows_held, ..) of this CTA into shared memory; every thread waits for
  // what it has copied itself, and masks it.
  auto fetch = [&](int b) {
    const int first = b * p.rows_held, n = min(n_rows - first, p.rows_held);
    const T* src = x + (int64_t)(first + lane_r) * p.ldx + (n_valid > 0 ? c : 0);
    uint32_t dst = own_s;
    if (p.wide) {
      for (int r = lane_r; r < n; r += RPP, dst += kPass, src += pass_elems)
        sm100::cp_async_16(dst, src, (uint32_t)(n_valid * (int)sizeof(T)));
    } else {
      for (int r = lane_r; r < n; r += RPP, dst += kPass, src += pass_elems) {
        const Vec<T> v = load_vec<T>(src, n_valid, false);
        sm100::st_shared_v4(dst, v.w[0], v.w[1], v.w[2], v.w[3]);
      }
    }
    sm100::cp_async_wait_all();
    if constexpr (DROP) {
      uint32_t at = own_s;
      for (int r = lane_r; r < n; r += RPP, at += kPass) {
        const uint4 u = sm100::ld_shared_v4(at);
        Vec<T> v;
        v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
        drop_vec<T>(p.drop, key, drop_index(p.drop, row0 + first + r, c), v);
        sm100::st_shared_v4(at, v.w[0], v.w[1], v.w[2], v.w[3]);
      }
    }
  };

  // Maxima and sums of this thread's V columns over the rows it has copied itself.
  uint32_t top[4];
  float sum[V];
#pragma unroll
  for (int j = 0; j < 4; ++j) top[j] = 0u;
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.f;
  const int batches = max(1, (n_rows + p.rows_held - 1) / max(1, p.rows_held));
  for (int b = 0; b < batches; ++b) {
    fetch(b);
    const int n = min(n_rows - b * p.rows_held, p.rows_held);
    uint32_t at = own_s;
    for (int r = lane_r; r < n; r += RPP, at += kPass) {
      const uint4 u = sm100::ld_shared_v4(at);
      Vec<T> v;
      v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) top[j] = max(top[j], v.w[j] & 0x7FFFFFFFu);
        else top[j] = __vmaxu2(top[j], v.w[j] & 0x7FFF7FFFu);
      }
      if (p.col_sums) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += v.get(j);
      }
    }
  }
  // Lanes lane % LANES of a warp hold the same columns.
#pragma unroll
  for (int s = LANES; s < 32; s *= 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t o = __shfl_xor_sync(0xFFFFFFFFu, top[j], s);
      top[j] = sizeof(T) == 4 ? max(top[j], o) : __vmaxu2(top[j], o);
    }
    if (p.col_sums) {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += __shfl_xor_sync(0xFFFFFFFFu, sum[j], s);
    }
  }
  if (lane < LANES) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      part_max[warp][lane * V + j] =
          sizeof(T) == 4 ? top[j & 3] : abs_bits_to_f32<T>(j & 1 ? top[(j / 2) & 3] >> 16 : top[(j / 2) & 3] & 0xFFFFu);
      part_sum[warp][lane * V + j] = sum[j];
    }
  }
  __syncthreads();
  if (threadIdx.x < COLS) {
    uint32_t m = 0;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kColWarps; ++w) {
      m = max(m, part_max[w][threadIdx.x]);
      s += part_sum[w][threadIdx.x];
    }
    cta_max[threadIdx.x] = m;
    cta_sum[threadIdx.x] = s;
  }
  __syncwarp();
  cluster.sync();
  // One thread per column combines the peers' results.
  if (threadIdx.x < COLS) {
    uint32_t m = 0;
    float s = 0.f;
    for (int i = 0; i < peers; ++i) {
      m = max(m, cluster.map_shared_rank(cta_max, i)[threadIdx.x]);
      if (rank == 0 && p.col_sums) s += cluster.map_shared_rank(cta_sum, i)[threadIdx.x];
    }
    const RowScale q = row_scale(m);
    scales[threadIdx.x] = q;
    const int64_t col = col0 + threadIdx.x;
    if (rank == 0 && col < p.cols) {
      const float grow = DROP ? p.drop.grow : 1.f;
      p.scale[col] = q.scale * grow;
      if (p.col_sums) p.col_sums[col] = s * grow;
    }
  }
  __syncthreads();
  sm100::cluster_arrive_relaxed();   // this CTA has read its peers' results; waited for at the end
  const int pair = lane % PAIRS, set = lane / PAIRS;
  const RowScale q0 = scales[2 * pair], q1 = scales[2 * pair + 1];
  const RowScale2 q01(q0, q1);
  const int64_t c0 = col0 + 2 * pair;
  // The last batch is still in shared memory; earlier ones are read again (from L2).
  for (int b = batches - 1; b >= 0; --b) {
    const int first = b * p.rows_held, n = min(n_rows - first, p.rows_held);
    if (b + 1 < batches) {
      __syncthreads();
      fetch(b);
      __syncthreads();
    }
    constexpr int kStep = kColWarps * SETS * 16;     // rows that the block rounds at once
    uint32_t at = held_s + (uint32_t)(held_at((warp * SETS + set) * 16) + pair * 2 * (int)sizeof(T));
    uint8_t* qa = p.q + c0 * p.ldq + row0 + first + (warp * SETS + set) * 16;
    for (int g = (warp * SETS + set) * 16; g < n; g += kStep, at += kStep / 16 * 17 * kStripBytes, qa += kStep) {
      uint32_t w0[4], w1[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t b0[4], b1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f0, f1;
          if constexpr (sizeof(T) == 4) {
            const uint2 u = sm100::ld_shared_v2(at + (uint32_t)((4 * k + j) * kStripBytes));
            f0 = __uint_as_float(u.x);
            f1 = __uint_as_float(u.y);
          } else {
            Vec<T> v;
            v.w[0] = sm100::ld_shared_u32(at + (uint32_t)((4 * k + j) * kStripBytes));
            f0 = v.get(0);
            f1 = v.get(1);
          }
          quantize_two<T>(f0, f1, q01, b0[j], b1[j]);
        }
        w0[k] = q0.c == 0.f ? 0u : pack4(b0[0], b0[1], b0[2], b0[3]);
        w1[k] = q1.c == 0.f ? 0u : pack4(b1[0], b1[1], b1[2], b1[3]);
      }
      auto store = [&](int64_t col, uint8_t* q, const uint32_t (&w)[4]) {
        if (col >= p.cols) return;
        if (n - g >= 16) {
          *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (g + j < n) q[j] = (uint8_t)(w[j / 4] >> (8 * (j & 3)));
        }
      };
      store(c0, qa, w0);
      store(c0 + 1, qa + p.ldq, w1);
    }
  }
  __syncwarp();                      // sets of a warp end at different rows; the wait needs all its lanes together
  sm100::cluster_wait();             // until the peers have read this CTA's
}

// ----------------------------------------------------------------- host
template <typename T, int NV, bool DROP>
cudaError_t launch_rows(const QuantParams& p, cudaStream_t st) {
  const int64_t nvec = (p.cols + Vec<T>::N - 1) / Vec<T>::N;
  int64_t tx = (nvec + NV - 1) / NV;
  tx = (tx + 31) / 32 * 32;
  if (tx > row_threads(NV)) tx = row_threads(NV);
  const int ry = tx >= 128 ? 1 : (int)(128 / tx);
  const int64_t blocks = (p.rows + ry - 1) / ry;   // at most 2^30
  return launch_overlapped(quantize_rows_kernel<T, NV, DROP>, dim3((unsigned)blocks), dim3((unsigned)tx, (unsigned)ry), 0, 1, st, p);
}
// Many loads in flight per thread for large X; two where one wave of threads covers
// it (333 x 1000 fp32 1.9 us, 3.7 with eight; 16384 x 8192 bf16 99 us, 70 with eight).  The
// mask's words need registers: four with dropout.
template <typename T>
cudaError_t launch_rows(const QuantParams& p, cudaStream_t st) {
  const int64_t nvec = (p.cols + Vec<T>::N - 1) / Vec<T>::N;
  if (p.rows * nvec <= 148 * 2048 && nvec <= 2 * row_threads(2))
    return p.drop.on ? launch_rows<T, 2, true>(p, st) : launch_rows<T, 2, false>(p, st);
  return p.drop.on ? launch_rows<T, 4, true>(p, st) : launch_rows<T, 8, false>(p, st);
}

template <typename T, bool DROP, int kColWarps>
cudaError_t launch_cols(QuantParams p, int peers, cudaStream_t st) {
  constexpr int kCols = kStripBytes / (int)sizeof(T);
  constexpr int kHeld = rows_held(DROP);
  p.rows_held = p.row_chunk < kHeld ? p.row_chunk : kHeld;
  const int64_t strips = (p.cols + kCols - 1) / kCols;
  const auto fn = quantize_cols_kernel<T, DROP, kColWarps>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld / 16 * 17 * kStripBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(fn, dim3((unsigned)(strips * peers)), dim3(32 * kColWarps),
                           (size_t)(p.rows_held / 16 * 17 * kStripBytes), peers, st, p);
}
// Four warps per CTA start sooner and leave room for more CTAs; eight pay off for CTAs
// with many rows (1024 x 8192 bf16 9.8 us and 11.4; with dropout and sums 16384 x 8192 272 us and 247).
template <typename T>
cudaError_t launch_cols(QuantParams p, cudaStream_t st) {
  int peers = (int)((p.rows + 255) / 256);
  peers = peers < 1 ? 1 : (peers > 8 ? 8 : peers);
  p.row_chunk = (int32_t)(((p.rows + peers - 1) / peers + 15) / 16 * 16);
  if (p.drop.on) return p.row_chunk <= 512 ? launch_cols<T, true, 4>(p, peers, st) : launch_cols<T, true, 8>(p, peers, st);
  return p.row_chunk <= 1024 ? launch_cols<T, false, 4>(p, peers, st) : launch_cols<T, false, 8>(p, peers, st);
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
