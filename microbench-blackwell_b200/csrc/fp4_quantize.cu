// fp4_quantize.cu -- rows of a floating matrix to 4-bit operands (fp4_common.cuh) and back.  Both are bound by
// the bytes of the floating side: 2 or 4 an element against 0.56.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "fp4_common.cuh"
#include "gemm_sm100a.h"
#include "row_stream.cuh"
#include "sm100_ptx.cuh"

using namespace int8op;
using namespace rowstream;

namespace {

struct QuantParams {
  const void* x;
  int64_t ldx, rows, cols;
  uint8_t* values;
  int64_t ldv;
  uint8_t* scales;
  int64_t tiles;
  float* row_scale;
  int32_t stages;              // rows ahead, and bytes of a stretch in shared memory (row_stream.cuh)
  uint32_t place;
};

// Few or very long rows.  A row belongs to blockDim.x threads (a block holds blockDim.y rows); each keeps NU units in
// registers between the row's maximum and the rounding, so X is read once.  Longer rows are read
// again (from L2) chunk by chunk.
template <typename T, int BLOCK, int NU>
__global__ void __launch_bounds__(512) quantize_fp4_kernel(const __grid_constant__ QuantParams p) {
  __shared__ uint32_t warp_max[16];
  const int tx = threadIdx.x, TX = blockDim.x;
  const int units = (int)(p.tiles * 4 * (BLOCK / 16));        // those of whole atoms of K: their scales are stored too
  const int per_chunk = NU * TX;
  const int chunks = (units + per_chunk - 1) / per_chunk;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const T* const x = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
  const int cols = live ? (int)p.cols : 0;
  rowvec::Unit<T> v[NU];
  auto load = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int e = (chunk * per_chunk + i * TX + tx) * kUnit;
      v[i] = rowvec::load_unit<T>(x + e, cols - e);
    }
  };
  uint32_t top = 0, tops[NU];   // largest |x| of the row, and of each unit held
  for (int c = 0; c < chunks; ++c) {
    load(c);
#pragma unroll
    for (int i = 0; i < NU; ++i) top = max(top, tops[i] = rowvec::magnitude(v[i]));
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (TX > 32) {
    const int warp = threadIdx.y * (TX >> 5) + (tx >> 5);
    if ((tx & 31) == 0) warp_max[warp] = top;
    __syncthreads();
    const int w = tx & 31;
    top = __reduce_max_sync(0xFFFFFFFFu, w < (TX >> 5) ? warp_max[threadIdx.y * (TX >> 5) + w] : 0u);
  }
  const fp4op::RowScale s = fp4op::row_scale(top);
  if (live && tx == 0) p.row_scale[row] = s.scale;
  const bool far = s.far();
  const float up = far ? 1.f : s.up, g = far ? 1.f : s.scale;
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int unit = c * per_chunk + i * TX + tx;
      if ((unit & ~31) >= units) break;      // whole warps
      if (chunks > 1) tops[i] = rowvec::magnitude(v[i]);
      float x[16], most = __uint_as_float(tops[i]);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = v[i].get(j);
      if (far) fp4op::bring_near(x, most, s);
      uint32_t q[2];
      const uint32_t code = fp4op::quantize_unit<BLOCK>(x, most, up, g, q);
      fp4op::store_scale_codes<BLOCK>(p.scales, row, p.tiles, unit, code, live && unit < units);
      const int n = cols - unit * kUnit;
      if (n > 0) fp4op::store_codes(p.values + row * p.ldv + unit * 8, q, n);
    }
  }
}

// Many rows: groups of threads walk down the matrix, NU units to a thread, with the coming rows copied ahead.
// 16384 x 8192 bf16 in 62 us (5.5 TB/s; the form above 110), fp32 101 (6.0 TB/s); issue slots are 65 % busy.
template <typename T, int BLOCK, int NU, bool FULL>
__global__ void __launch_bounds__(NU == 2 ? 768 : 512, 1) quantize_fp4_stream_kernel(const __grid_constant__ QuantParams p) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ uint32_t warp_max[2][32];
  constexpr int E = (int)sizeof(T);
  const int tx = threadIdx.x, TX = blockDim.x, warps = TX >> 5;
  const int units = (int)(p.tiles * 4 * (BLOCK / 16));
  const uint32_t per_stage = NU * p.place;
  const uint32_t mine = sm100::smem_u32(slots) + (uint32_t)((int)threadIdx.y * warps + (tx >> 5)) * (uint32_t)p.stages * per_stage;
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, step = (int64_t)gridDim.x * blockDim.y;
  int n[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) n[i] = (int)p.cols - (i * TX + tx) * kUnit;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  auto issue = [&](int64_t row, uint32_t slot) {
    if (row < p.rows) {
      const uint8_t* const r = row_of(static_cast<const uint8_t*>(p.x), row, p.ldx * E) + (tx & ~31) * kUnit * E;
#pragma unroll
      for (int i = 0; i < NU; ++i) issue_stretch<T, FULL>(slot + i * p.place, r + i * TX * kUnit * E, n[i] + (tx & 31) * kUnit);
    }
    commit_copies();
  };
  for (int s = 0; s < p.stages; ++s) issue(first + s * step, mine + (uint32_t)s * per_stage);
  int stage = 0, flip = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const uint32_t at = mine + (uint32_t)stage * per_stage;
    wait_copies(p.stages - 1);
    __syncwarp();
    const uint32_t off = FULL ? 0u : (uint32_t)reinterpret_cast<uintptr_t>(static_cast<const uint8_t*>(p.x) + row * p.ldx * E) & 15u;
    Unit<T> v[NU];
    uint32_t tops[NU], top = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      v[i] = take_unit<T, FULL>(at + i * p.place, off, n[i]);
      top = max(top, tops[i] = rowvec::magnitude(v[i]));
    }
    __syncwarp();
    issue(row + p.stages * step, at);
    if (++stage == p.stages) stage = 0;
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (warps > 1) {
      // (A row's maxima are written again by the second row after it, with a barrier between.)
      uint32_t* const group = warp_max[flip ^= 1] + (int)threadIdx.y * warps;
      if ((tx & 31) == 0) group[tx >> 5] = top;
      group_sync();
      top = __reduce_max_sync(0xFFFFFFFFu, (tx & 31) < warps ? group[tx & 31] : 0u);
    }
    const fp4op::RowScale s = fp4op::row_scale(top);
    if (tx == 0) p.row_scale[row] = s.scale;
    const bool far = s.far();
    const float up = far ? 1.f : s.up, g = far ? 1.f : s.scale;
    uint8_t* const out = row_of(p.values, row, p.ldv);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int unit = i * TX + tx;
      if ((unit & ~31) >= units) break;      // whole warps
      forget(v[i]);
      float x[16], most = __uint_as_float(tops[i]);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = v[i].get(j);
      if (each_row(far)) fp4op::bring_near(x, most, s);
      uint32_t q[2];
      const uint32_t code = fp4op::quantize_unit<BLOCK>(x, most, up, g, q);
      fp4op::store_scale_codes<BLOCK>(p.scales, row, p.tiles, unit, code, unit < units);
      if (n[i] > 0) fp4op::store_codes(out + unit * 8, q, n[i]);
    }
  }
}

template <typename T, int BLOCK, int NU>
cudaError_t launch_rows(const QuantParams& p, cudaStream_t st) {
  const int64_t units = p.tiles * 4 * (BLOCK / 16);
  int64_t tx = ((units + NU - 1) / NU + 31) / 32 * 32;
  if (tx > 512) tx = 512;
  const int ry = tx >= 128 ? 1 : (int)(128 / tx);
  const int64_t blocks = (p.rows + ry - 1) / ry;   // at most 2^30
  return launch_overlapped(quantize_fp4_kernel<T, BLOCK, NU>, dim3((unsigned)blocks), dim3((unsigned)tx, (unsigned)ry), 0, 1, st, p);
}
template <typename T, int BLOCK, int NU, bool FULL>
cudaError_t launch_stream(QuantParams p, cudaStream_t st) {
  p.place = place_bytes((int)sizeof(T), FULL || all_wide({{p.x, p.ldx * (int64_t)sizeof(T)}}));
  const Shape s = shape_of(p.rows, (int)(p.tiles * 4 * (BLOCK / 16)), NU, NU * (int)p.place, NU == 2 ? 768 : 512);
  if (s.stages < 1) return cudaErrorInvalidValue;
  p.stages = s.stages;
  const auto fn = quantize_fp4_stream_kernel<T, BLOCK, NU, FULL>;
  const cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (err != cudaSuccess) return err;
  return launch_overlapped(fn, dim3((unsigned)s.blocks), dim3((unsigned)s.tx, (unsigned)s.ty), s.smem, 1, st, p);
}
template <typename T, int BLOCK>
cudaError_t launch_rows(const QuantParams& p, cudaStream_t st) {
  const int64_t units = p.tiles * 4 * (BLOCK / 16);
  // One unit to a thread where a wave of threads covers X: one row of 8192 in 1.8 us.
  if (p.rows * units <= 148 * 1024) return launch_rows<T, BLOCK, 1>(p, st);
  if (units > 4 * kMaxThreads) return launch_rows<T, BLOCK, 2>(p, st);
  const bool wide = all_wide({{p.x, p.ldx * (int64_t)sizeof(T)}}) && p.cols < INT32_MAX / 2 &&
                    all_full((int)units, (int)p.cols, units <= 2 * kMaxThreads ? 2 : 4);
  if (units <= 2 * kMaxThreads) return wide ? launch_stream<T, BLOCK, 2, true>(p, st) : launch_stream<T, BLOCK, 2, false>(p, st);
  return wide ? launch_stream<T, BLOCK, 4, true>(p, st) : launch_stream<T, BLOCK, 4, false>(p, st);
}
template <typename T>
cudaError_t launch_rows(const QuantParams& p, int block, cudaStream_t st) {
  return block == 16 ? launch_rows<T, 16>(p, st) : launch_rows<T, 32>(p, st);
}

// ----------------------------------------------------------------- back
struct DequantParams {
  const uint8_t* values;
  int64_t ldv, rows, cols;
  const uint8_t* scales;
  int64_t tiles;
  const float* row_scale;
  void* y;
  int64_t ldy;
};

// value * scale has at most seven bits; a row scale that is a power of two keeps it exact within fp32's range.
// A thread takes a unit of a column of units, two rows at a time.
template <typename T, int BLOCK>
__global__ void __launch_bounds__(256) dequantize_fp4_kernel(const __grid_constant__ DequantParams p) {
  constexpr int UN = 2;
  const int unit = (int)blockIdx.x * (int)blockDim.x + (int)threadIdx.x;
  const int e = unit * kUnit;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const int n = (int)min((int64_t)kUnit, p.cols - e);
  const int64_t step = (int64_t)gridDim.y * blockDim.y;
  for (int64_t row0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row0 < p.rows; row0 += UN * step) {
    uint32_t q[UN][2], code[UN];
    float g[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t row = row0 + u * step;
      q[u][0] = q[u][1] = code[u] = 0u;
      g[u] = 1.f;
      if (n > 0 && row < p.rows) {
        const uint8_t* const at = p.values + row * p.ldv + unit * 8;
        if (n == kUnit && (reinterpret_cast<uintptr_t>(at) & 7) == 0) {
          const uint2 w = *reinterpret_cast<const uint2*>(at);
          q[u][0] = w.x;
          q[u][1] = w.y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (2 * j < n) q[u][j / 4] |= (uint32_t)at[j] << (8 * (j & 3));
        }
        code[u] = p.scales[fp4op::scale_at(row, unit / (BLOCK / 16), p.tiles)];
        if (p.row_scale) g[u] = p.row_scale[row];
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t row = row0 + u * step;
      if (row >= p.rows) break;          // (whole warps)
      const float s = BLOCK == 16 ? fp4op::decode_e4m3(code[u]) : fp4op::decode_e8m0(code[u]);
      rowvec::Unit<T> o;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t h;
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}"
            : "=r"(h) : "r"(q[u][j / 4] >> (8 * (j & 3))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        o.set2(2 * j, f.x * s * g[u], f.y * s * g[u]);
      }
      rowvec::store_unit<T>(static_cast<T*>(p.y) + row * p.ldy + e, o, n);
    }
  }
}

template <typename T>
cudaError_t launch_back(const DequantParams& p, int block, cudaStream_t st) {
  const int64_t units = (p.cols + kUnit - 1) / kUnit;
  const int64_t gx = (units + 255) / 256;
  const int tx = (int)(((units + gx - 1) / gx + 31) / 32 * 32);      // even parts of the row
  const int ty = 256 / tx;
  int64_t gy = (p.rows + ty - 1) / ty;
  const int64_t most = (148 * 32 + gx - 1) / gx;
  if (gy > most) gy = most;
  if (gy > 65535) gy = 65535;
  return launch_overlapped(block == 16 ? dequantize_fp4_kernel<T, 16> : dequantize_fp4_kernel<T, 32>, dim3((unsigned)gx, (unsigned)gy),
                           dim3((unsigned)tx, (unsigned)ty), 0, 1, st, p);
}

bool sizes_ok(int type, int64_t rows, int64_t cols, int block) {
  return type_ok(type) && fp4op::block_ok(block) && rows >= 0 && cols >= 0 && rows <= INT32_MAX / 2 && cols <= INT32_MAX / 2;
}
int status_of(cudaError_t err) {
  if (err == cudaSuccess) return GEMM_OK;
  cudaGetLastError();
  return GEMM_ERR_LAUNCH;
}

}  // namespace

extern "C" int64_t gemm_sm100a_fp4_scale_bytes(int64_t rows, int64_t cols, int32_t block) {
  if (!sizes_ok(GEMM_TYPE_BF16, rows, cols, block)) return -1;
  return (rows + 127) / 128 * fp4op::scale_tiles(cols, block) * 512;
}

extern "C" int gemm_sm100a_quantize_fp4(const Fp4QuantArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(Fp4QuantArgs)) return GEMM_ERR_BAD_ARGS;
  if (!sizes_ok(a->x_type, a->rows, a->cols, a->block)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->rows == 0 || a->cols == 0) return GEMM_OK;
  if (!a->x || !a->values || !a->scales || !a->row_scale) return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->x_type);
  if (a->ldx < a->cols || reinterpret_cast<uintptr_t>(a->x) % e != 0 || a->ldv < (a->cols + 1) / 2 || a->ldv % 16 != 0 ||
      ((reinterpret_cast<uintptr_t>(a->values) | reinterpret_cast<uintptr_t>(a->scales)) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(a->row_scale) & 3) != 0)
    return GEMM_ERR_CANNOT_IMPLEMENT;
  QuantParams p;
  memset(&p, 0, sizeof(p));
  p.x = a->x; p.ldx = a->ldx; p.rows = a->rows; p.cols = a->cols;
  p.values = static_cast<uint8_t*>(a->values); p.ldv = a->ldv;
  p.scales = static_cast<uint8_t*>(a->scales); p.tiles = fp4op::scale_tiles(a->cols, a->block);
  p.row_scale = a->row_scale;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->values);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  return status_of(a->x_type == GEMM_TYPE_BF16 ? launch_rows<__nv_bfloat16>(p, a->block, st)
                 : a->x_type == GEMM_TYPE_FP16 ? launch_rows<__half>(p, a->block, st) : launch_rows<float>(p, a->block, st));
}

extern "C" int gemm_sm100a_dequantize_fp4(const Fp4DequantArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(Fp4DequantArgs)) return GEMM_ERR_BAD_ARGS;
  if (!sizes_ok(a->y_type, a->rows, a->cols, a->block)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->rows == 0 || a->cols == 0) return GEMM_OK;
  if (!a->y || !a->values || !a->scales) return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->y_type);
  if (a->ldy < a->cols || reinterpret_cast<uintptr_t>(a->y) % e != 0 || a->ldv < (a->cols + 1) / 2 ||
      (reinterpret_cast<uintptr_t>(a->row_scale) & 3) != 0)
    return GEMM_ERR_CANNOT_IMPLEMENT;
  DequantParams p;
  memset(&p, 0, sizeof(p));
  p.values = static_cast<const uint8_t*>(a->values); p.ldv = a->ldv; p.rows = a->rows; p.cols = a->cols;
  p.scales = static_cast<const uint8_t*>(a->scales); p.tiles = fp4op::scale_tiles(a->cols, a->block);
  p.row_scale = a->row_scale; p.y = a->y; p.ldy = a->ldy;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->y);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  return status_of(a->y_type == GEMM_TYPE_BF16 ? launch_back<__nv_bfloat16>(p, a->block, st)
                 : a->y_type == GEMM_TYPE_FP16 ? launch_back<__half>(p, a->block, st) : launch_back<float>(p, a->block, st));
}
