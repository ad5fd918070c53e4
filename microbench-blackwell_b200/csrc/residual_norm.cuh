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
// s + x^2 for the 64-bit number x with these upper 32 bits and zeros below them.
__device__ __forceinline__ void add_square(double& s, uint32_t upper) {
  asm volatile("{\n\t.reg .f64 x;\n\tmov.b64 x, {%2, %1};\n\tfma.rn.f64 %0, x, x, %0;\n\t}" : "+d"(s) : "r"(upper), "r"(0));
}
// Sum of a thread's squares of 16-bit elements in 64 bits, as hi + lo, |lo| <= 2^-24 hi.  (In fp32 a row whose mean one
// channel makes up loses 2^-20 of it, and the last bit of r turns elements of x_out and codes of a 4-bit operand.)  The numbers are put
// together from the elements' bits, exponents moved by 896: conversions would take longer than all the rest
// (16384 x 8192 bf16: 333 us with them, 170 without; 193 with sums of paired fp32).  A zero or a subnormal bf16 counts as
// some 2^-127, whose square is nothing beside the least sum that is used (out_of_range).
template <typename T, int NU>
__device__ __forceinline__ void squares(const Unit<T> (&u)[NU], float& hi, float& lo) {
  double s0 = 0.0, s1 = 0.0;
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < Unit<T>::W; ++j) {
      if constexpr (std::is_same<T, __half>::value) {
        add_square(s0, (__float_as_uint(fabsf(u[i].get(2 * j))) >> 3) + 0x38000000u);
        add_square(s1, (__float_as_uint(fabsf(u[i].get(2 * j + 1))) >> 3) + 0x38000000u);
      } else {
        add_square(s0, ((u[i].w[j] & 0x7FFFu) << 13) + 0x38000000u);
        add_square(s1, ((u[i].w[j] & 0x7FFF0000u) >> 3) + 0x38000000u);
      }
    }
  const double s = s0 + s1;
  hi = (float)s;
  lo = (float)(s - (double)hi);
}
template <typename T>
__device__ __forceinline__ double squares_wide(const Unit<T>& u) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kUnit; ++j) s = fma((double)u.get(j), (double)u.get(j), s);
  return s;
}
// Where a sum of squares may have left its parts' range in fp32 (or come near its end), it is taken again, all in 64 bits.
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

// The same for parts hi + lo >= 0 as above, in whole numbers of 2^-50 of a unit that goes by the largest part: 25 bits of
// hi and what is left of it with lo, so that 2^-45 of the sum are lost, and the hardware's integer reductions take a fraction of the
// time of a tree of 64-bit shuffles.
// A NaN or an infinity gives NaN.
struct WarpSum {
  uint64_t sum;      // < 2^55
  uint32_t e;
};
__device__ __forceinline__ double group_sum_parts(float hi, float lo, WarpSum* part) {
  const int warps = (int)blockDim.x >> 5, lane = (int)(threadIdx.x & 31u);
  // hi + lo = (i + j / 2^25) 2^(e - 151)
  uint32_t e = max(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(hi)) >> 23, 24u);
  const float unit = __uint_as_float((278u - e) << 23), f = hi * unit;
  const uint32_t i = __float2uint_rn(f);
  const int j = __float2int_rn(fmaf(lo, unit, f - (float)i) * 0x1p25f);
  uint64_t sum = ((uint64_t)__reduce_add_sync(0xFFFFFFFFu, i) << 25) + (uint64_t)(int64_t)__reduce_add_sync(0xFFFFFFFFu, j);
  if (warps > 1) {
    WarpSum* const mine = part + threadIdx.y * warps;
    if (lane == 0) mine[threadIdx.x >> 5] = {sum, e};
    group_sync();
    const WarpSum w = lane < warps ? mine[lane] : WarpSum{0ull, 0u};
    e = __reduce_max_sync(0xFFFFFFFFu, w.e);
    sum = w.sum >> min(e - w.e, 63u);
    // At most 16 warps.
    const uint32_t up = __reduce_add_sync(0xFFFFFFFFu, (uint32_t)(sum >> 28)), low = __reduce_add_sync(0xFFFFFFFFu, (uint32_t)sum & 0xFFFFFFFu);
    sum = ((uint64_t)up << 28) + low;
  }
  if (e >= 255u) return __longlong_as_double(0x7FF8000000000000ll);
  return (double)sum * __hiloint2double((int)((e + 1023u - 176u) << 20), 0);
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
