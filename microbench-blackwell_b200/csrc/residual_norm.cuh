// residual_norm.cuh -- what the norms around a block and their gradients share: statistics of a row, the vectors.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_sm100a.h"
#include "row_stream.cuh"
#include "sm100_ptx.cuh"

namespace {

using namespace int8op;
using namespace rowstream;

constexpr int kMaxCols = 16384;

// ----------------------------------------------------------------- statistics
template <typename T>
__device__ __forceinline__ F2 pair(const Unit<T>& u, int j) { return F2(u.get(2 * j), u.get(2 * j + 1)); }
__device__ __forceinline__ float both(F2 v) {
  float a, b;
  v.get(a, b);
  return a + b;
}
__device__ __forceinline__ F2 f2(float v) { return F2(v, v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ float squares(const Unit<T>& u) {
  F2 s = f2(0.f);
#pragma unroll
  for (int j = 0; j < kUnit / 2; ++j) s = fma2(pair(u, j), pair(u, j), s);
  return both(s);
}
template <typename T>
__device__ __forceinline__ double squares_wide(const Unit<T>& u) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kUnit; ++j) s = fma((double)u.get(j), (double)u.get(j), s);
  return s;
}
// Where the fp32 part of a sum of squares may have left its range (or come near its end), 64 bits do it again.
__device__ __forceinline__ bool out_of_range(float s) { return !(s > 1e-30f && s < 1e38f); }

// 1 / sqrt(v), rounded to fp32 from an error of 2^-43 or so: one Newton step whose 1 - v r^2 has v and r^2 in two fp32
// words each.
__device__ __forceinline__ float inverse_root(double v) {
  if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
  const float hi = (float)v, lo = (float)(v - (double)hi);
  const float r = rsqrtf(hi), p = r * r, p_lo = fmaf(r, r, -p);
  const float t = fmaf(-hi, p, 1.f) - fmaf(hi, p_lo, lo * p);
  return fmaf(0.5f * r, t, r);
}

// The sum over the group's threads; all of them call, with `part` alternating between calls.
__device__ __forceinline__ double group_sum(double v, double* part) {
  v = warp_sum(v);
  const int warps = (int)blockDim.x >> 5, lane = (int)(threadIdx.x & 31u);
  if (warps == 1) return v;
  double* const mine = part + threadIdx.y * warps;
  if (lane == 0) mine[threadIdx.x >> 5] = v;
  group_sync();
  v = lane < warps ? mine[lane] : 0.0;
  // At most 16 warps.
#pragma unroll
  for (int o = 8; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return __shfl_sync(0xFFFFFFFFu, v, 0);
}

// The same for fp32 parts >= 0, in whole numbers of a unit that goes by the largest part: 25 bits of each, so some 2^-28 of the
// sum are lost, and the hardware's integer reductions take a fraction of the time of a tree of shuffles (16384 x 8192 bf16
// into a 4-bit operand: 235 us with shuffles of 64 bits, 223 with these).
// A NaN or an infinity gives NaN.
__device__ __forceinline__ double group_sum_parts(float f, uint2* part) {
  const int warps = (int)blockDim.x >> 5, lane = (int)(threadIdx.x & 31u);
  // f = i 2^(e - 151)
  uint32_t e = max(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(f)) >> 23, 24u);
  uint32_t t = __reduce_add_sync(0xFFFFFFFFu, __float2uint_rn(f * __uint_as_float((278u - e) << 23)));
  if (warps > 1) {
    uint2* const mine = part + threadIdx.y * warps;
    if (lane == 0) mine[threadIdx.x >> 5] = make_uint2(t, e);
    group_sync();
    const uint2 w = lane < warps ? mine[lane] : make_uint2(0u, 0u);
    e = __reduce_max_sync(0xFFFFFFFFu, w.y);
    const uint32_t down = min(4u + e - w.y, 31u);                             // at most 16 warps of less than 2^30
    t = __reduce_add_sync(0xFFFFFFFFu, (w.x + (1u << (down - 1u))) >> down);
    e += 4u;
  }
  if (e >= 255u) return __longlong_as_double(0x7FF8000000000000ll);
  return (double)t * __hiloint2double((int)((e + 1023u - 151u) << 20), 0);
}

// ----------------------------------------------------------------- vectors
// A vector's elements at a thread's unit as fp32 pairs; ones where there is no vector.
template <typename T>
__device__ __forceinline__ void load_params(const void* v, int param32, int e, int n, F2 (&o)[kUnit / 2]) {
  if (!v) {
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = f2(1.f);
  } else if (sizeof(T) == 4 || param32) {
    const Unit<float> u = rowvec::load_unit<float, rowvec::kKeep>(static_cast<const float*>(v) + e, n);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = pair(u, j);
  } else {
    const Unit<T> u = rowvec::load_unit<T, rowvec::kKeep>(static_cast<const T*>(v) + e, n);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = pair(u, j);
  }
}

// Vectors that all groups of a block read, in shared memory: four elements of a unit to a slot, the slots of one kind side by
// side for all units (no bank conflicts).
struct SharedVectors {
  uint32_t base, per_chunk;      // bytes from a unit's slot to that of its next four elements
  __device__ __forceinline__ uint32_t at(int which, int unit) const { return base + (uint32_t)(which * 4) * per_chunk + (uint32_t)unit * 16u; }
  __device__ __forceinline__ void put(int which, int unit, const F2 (&v)[kUnit / 2]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float f[4];
      v[2 * c].get(f[0], f[1]);
      v[2 * c + 1].get(f[2], f[3]);
      sm100::st_shared_v4(at(which, unit) + (uint32_t)c * per_chunk, __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
  }
  // Pairs 2 c and 2 c + 1 of a unit.
  __device__ __forceinline__ void get(int which, int unit, int c, F2& a, F2& b) const {
    const uint4 u = sm100::ld_shared_v4(at(which, unit) + (uint32_t)c * per_chunk);
    a = F2(__uint_as_float(u.x), __uint_as_float(u.y));
    b = F2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  __device__ __forceinline__ void get(int which, int unit, F2 (&v)[kUnit / 2]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) get(which, unit, c, v[2 * c], v[2 * c + 1]);
  }
};

// ----------------------------------------------------------------- host
int status_of(cudaError_t err) {
  if (err == cudaSuccess) return GEMM_OK;
  cudaGetLastError();
  return GEMM_ERR_LAUNCH;
}
bool aligned(const void* p, int e) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)e == 0; }

}  // namespace
