// int8_common.cuh -- what the 8-bit integer operators share: element types,
// the dropout mask, exact int8 rounding and host-side argument checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "counter_rng.cuh"
#include "gemm_sm100a.h"

namespace int8op {

__host__ __device__ constexpr int type_bytes(int t) { return t == GEMM_TYPE_FP32 ? 4 : 2; }
__host__ __device__ constexpr bool type_ok(int t) { return t >= GEMM_TYPE_BF16 && t <= GEMM_TYPE_FP32; }

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// Element i of a vector of run-time type t.
__device__ __forceinline__ float load_as_f32(const void* p, int t, int64_t i) {
  if (t == GEMM_TYPE_FP32) return static_cast<const float*>(p)[i];
  if (t == GEMM_TYPE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}

// One output of the product from its exact sum, before dropout and residual.
__device__ __forceinline__ float finish(int32_t acc, float sa, float sb, float bias) {
  return fmaf(__int2float_rn(acc) * sa, sb, bias);
}
// The sum times a larger scale than this might leave the range of fp32 (2^31 * 2^96 does not)
// where the output does not.  The channel's scale then comes first: only if it is as
// large too can that product overflow, and so does the output.
constexpr float kLargeScale = 0x1p96f;
__device__ __forceinline__ bool is_large(float sa) { return fabsf(sa) > kLargeScale; }
__device__ __forceinline__ float finish_large(int32_t acc, float sa, float sb, float bias) {
  const bool large = is_large(sa);
  return finish(acc, large ? sb : sa, large ? sa : sb, bias);
}

// Two 16-bit values, rounded, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float f0, float f1) {
  uint32_t u;
  if constexpr (sizeof(T) == 2) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(f0, f1);
      __builtin_memcpy(&u, &h, 4);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f0, f1);
      __builtin_memcpy(&u, &h, 4);
    }
  }
  return u;
}

// 16 bytes of T as registers; element access is compile-time indexed.
template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t h = (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu);
      T v;
      __builtin_memcpy(&v, &h, 2);
      return to_f32(v);
    }
  }
  // Elements i and i + 1 (i even), rounded.
  __device__ __forceinline__ void set2(int i, float f0, float f1) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(f0);
      w[i + 1] = __float_as_uint(f1);
    } else {
      w[i / 2] = pack2<T>(f0, f1);
    }
  }
  __device__ __forceinline__ void zero(int i) {
    if constexpr (sizeof(T) == 4) w[i] = 0u;
    else w[i / 2] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
  }
};

// Elements [0, n) of p (n <= Vec<T>::N; the rest reads as 0).  `wide`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, int n, bool wide) {
  Vec<T> v;
  if (n >= Vec<T>::N && wide) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
  } else {
    v.w[0] = v.w[1] = v.w[2] = v.w[3] = 0u;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4) {
          v.w[i] = __float_as_uint(reinterpret_cast<const float*>(p)[i]);
        } else {
          const uint32_t h = reinterpret_cast<const uint16_t*>(p)[i];
          v.w[i / 2] |= i & 1 ? h << 16 : h;
        }
      }
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v, int n, bool wide) {
  if (n >= Vec<T>::N && wide) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[i] = v.w[i];
        else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(i & 1 ? v.w[i / 2] >> 16 : v.w[i / 2] & 0xFFFFu);
      }
  }
}

// ------------------------------------------------------------------ dropout
// Kernel-side form of DropoutArgs.
struct Drop {
  uint64_t seed_mix;            // seed + mix64(stream_id + golden)
  const uint64_t* seed_offset;
  uint32_t threshold;           // a word below rint(p * 2^32) is dropped (unless `all`: at least 1)
  float grow;                   // 1 / (1 - p), 0 for p = 1
  int32_t on;
  int32_t all;                  // p rounds to 1 in steps of 2^-32: every element is dropped
  int64_t row0, col0, row_elems;
};

__device__ __forceinline__ uint64_t drop_key(const Drop& d) {
  return counter_rng::mix64(d.seed_mix + (d.seed_offset ? *d.seed_offset : 0ull));
}
__device__ __forceinline__ int64_t drop_index(const Drop& d, int64_t r, int64_t c) {
  return (d.row0 + r) * d.row_elems + d.col0 + c;
}
__device__ __forceinline__ bool drop_keeps(const Drop& d, uint64_t key, int64_t index) {
  const uint64_t h = counter_rng::draw(key, (uint64_t)index >> 1);
  return !d.all && (uint32_t)(index & 1 ? h >> 32 : h) >= d.threshold;
}
// The words of elements `index` .. + N - 1 (N even); zeros where all are dropped.
// One draw serves the two elements of an aligned pair.
template <int N>
__device__ __forceinline__ void drop_words(const Drop& d, uint64_t key, int64_t index, uint32_t (&w)[N]) {
  uint64_t z = key + (((uint64_t)index >> 1) + 1) * counter_rng::kGolden;
#pragma unroll
  for (int j = 0; j < N / 2; ++j, z += counter_rng::kGolden) {
    const uint64_t h = counter_rng::mix64(z);
    w[2 * j] = (uint32_t)h;
    w[2 * j + 1] = (uint32_t)(h >> 32);
  }
  if (index & 1) {
    const uint64_t h = counter_rng::mix64(z);
#pragma unroll
    for (int j = 0; j + 1 < N; ++j) w[j] = w[j + 1];
    w[N - 1] = (uint32_t)h;
  }
  if (d.all) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = 0u;
  }
}

// Zeroes the dropped elements of a vector that starts at element `index`.
template <typename T>
__device__ __forceinline__ void drop_vec(const Drop& d, uint64_t key, int64_t index, Vec<T>& v) {
  uint32_t w[Vec<T>::N];
  drop_words<Vec<T>::N>(d, key, index, w);
  const uint32_t threshold = d.threshold;
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j)
    if (w[j] < threshold) v.zero(j);
}
// ------------------------------------------------------------------ int8 rounding
// q = 127 * x / amax to the nearest integer, ties to even, decided exactly.
// Everything is scaled by a power of two g so that neither the products nor
// the reciprocal leave the normal range.
constexpr float kAmaxMin = 127.0f * 1.17549435e-38f;   // 127 * 2^-126

struct RowScale {
  float c;      // 127 * g, 0 for a row with NaN or Inf
  float a;      // amax * g
  float ra;     // 1 / a
  float scale;  // amax / 127
};

// `bits`: the largest |x| of the row as fp32 bits (integer maximum, so NaN > Inf > finite).
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale s;
  if (bits >= 0x7F800000u) {
    s.c = 0.f; s.a = 1.f; s.ra = 1.f; s.scale = __uint_as_float(bits);
    return s;
  }
  const float amax = fmaxf(__uint_as_float(bits), kAmaxMin);
  const float g = amax < 0x1p-60f ? 0x1p64f : (amax > 0x1p60f ? 0x1p-64f : 1.f);
  s.c = 127.f * g;
  s.a = amax * g;
  s.ra = __frcp_rn(s.a);
  s.scale = __fdiv_rn(amax, 127.f);
  return s;
}

constexpr float kRound = 12582912.f;   // 1.5 * 2^23: adding it leaves the nearest integer in the low byte

// Low byte: q of an element.
//  16-bit x: 127 x g is exact in fp32 and one correction step gives the
//    quotient t to one unit in the last place, exactly where it is a tie.  With
//    significands of 18 and 11 bits a t >= 1/4 that is not half-way between
//    integers is at least 2^-20 t away from there, 16 times that error.
//  fp32 x: f is an integer with f - eps <= t <= f + 1 + eps for the quotient t;
//    the sign of 127 x g - a (f + 1/2), whose first term is held as yh + yl and
//    whose fused difference is exact near zero, says whether t rounds to f + 1.
// Two elements at a time, each with its row's scale, in packed fp32 operations.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
struct RowScale2 {
  F2 c, na, ra;   // 127 * g, -amax * g, 1 / (amax * g) of both
  __device__ __forceinline__ RowScale2(const RowScale& s0, const RowScale& s1) : c(s0.c, s1.c), na(-s0.a, -s1.a), ra(s0.ra, s1.ra) {}
};

template <typename T>
__device__ __forceinline__ void quantize_two(float x0, float x1, const RowScale2& s, uint32_t& q0, uint32_t& q1) {
  const F2 x(x0, x1), round(kRound, kRound);
  const F2 y = mul2(x, s.c);
  float m0, m1;
  if constexpr (sizeof(T) == 2) {
    const F2 t = mul2(y, s.ra);
    const F2 r = fma2(s.na, t, y);
    add2(fma2(r, s.ra, t), round).get(m0, m1);
    q0 = __float_as_uint(m0);
    q1 = __float_as_uint(m1);
  } else {
    float y0, y1, d0, d1;
    y.get(y0, y1);
    const F2 yl = fma2(x, s.c, F2(-y0, -y1));
    const F2 m = add2(fma2(y, s.ra, F2(-0.5f, -0.5f)), round);
    const F2 f = add2(m, F2(-kRound, -kRound));
    add2(fma2(s.na, add2(f, F2(0.5f, 0.5f)), y), yl).get(d0, d1);
    m.get(m0, m1);
    q0 = __float_as_uint(m0);
    q1 = __float_as_uint(m1);
    // d > 0, or a tie (d = 0) above an odd f: d above the largest negative number or above zero.
    q0 += d0 > __uint_as_float((q0 & 1u) * 0x80000001u) ? 1u : 0u;
    q1 += d1 > __uint_as_float((q1 & 1u) * 0x80000001u) ? 1u : 0u;
  }
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Magnitude bits of a T as fp32 bits.
template <typename T>
__device__ __forceinline__ uint32_t abs_bits_to_f32(uint32_t h) {
  if constexpr (sizeof(T) == 4) return h;
  else {
    const uint16_t u = (uint16_t)h;
    T v;
    __builtin_memcpy(&v, &u, 2);
    return __float_as_uint(to_f32(v));
  }
}

// Largest |x| of a vector as fp32 bits.
template <typename T>
__device__ __forceinline__ uint32_t vec_magnitude(const Vec<T>& v) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) m = max(m, v.w[j] & 0x7FFFFFFFu);
    else m = __vmaxu2(m, v.w[j] & 0x7FFF7FFFu);
  }
  if constexpr (sizeof(T) == 2) m = abs_bits_to_f32<T>(max(m & 0xFFFFu, m >> 16));
  return m;
}
// The int8 values of a vector, four to a word.
template <typename T>
__device__ __forceinline__ void quantize_vec(const Vec<T>& v, const RowScale& s, uint32_t (&w)[Vec<T>::N / 4]) {
  const RowScale2 s2(s, s);
#pragma unroll
  for (int j = 0; j < Vec<T>::N / 4; ++j) {
    uint32_t q[4];
    quantize_two<T>(v.get(4 * j), v.get(4 * j + 1), s2, q[0], q[1]);
    quantize_two<T>(v.get(4 * j + 2), v.get(4 * j + 3), s2, q[2], q[3]);
    w[j] = s.c == 0.f ? 0u : pack4(q[0], q[1], q[2], q[3]);
  }
}

// ------------------------------------------------------------------ host
// Launch a kernel that begins with grid_dependency_wait(): its launch latency
// overlaps the end of the kernel before it.
template <typename... P, typename... A>
cudaError_t launch_overlapped(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, args...);
}

inline int drop_resolve(const DropoutArgs& a, int64_t rows, int64_t cols, Drop& d, const char** why) {
  d = Drop{};
  if (!(a.p >= 0.0 && a.p <= 1.0)) { *why = "dropout p must be in [0, 1]"; return GEMM_ERR_CANNOT_IMPLEMENT; }
  if (a.p == 0.0) return GEMM_OK;
  if (a.row0 < 0 || a.col0 < 0) { *why = "dropout row0/col0 must be >= 0"; return GEMM_ERR_CANNOT_IMPLEMENT; }
  if (a.row_elems < cols || a.col0 > a.row_elems - cols) {
    *why = "dropout row_elems must be >= col0 + columns";
    return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  if (((__int128)a.row0 + rows) * a.row_elems > ((__int128)1 << 62)) {
    *why = "dropout index beyond 2^62";
    return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  if (reinterpret_cast<uintptr_t>(a.seed_offset) & 7) {
    *why = "dropout seed_offset must be 8-byte aligned";
    return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  d.on = 1;
  d.seed_mix = a.seed + counter_rng::mix64(a.stream_id + counter_rng::kGolden);
  d.seed_offset = a.seed_offset;
  const uint64_t threshold = (uint64_t)std::llrint(a.p * 4294967296.0);
  d.all = threshold >> 32 ? 1 : 0;
  d.threshold = d.all ? 1u : (uint32_t)threshold;
  d.grow = a.p == 1.0 ? 0.f : (float)(1.0 / (1.0 - a.p));
  d.row0 = a.row0; d.col0 = a.col0; d.row_elems = a.row_elems;
  return GEMM_OK;
}

// Whether two matrices of `rows` rows each (at least one; lengths and strides in bytes) share a byte; also
// where a stride is shorter than its rows and the extents cross.  Matrices side by side in one buffer do not, though their extents cross.
inline bool rows_meet(const void* p, int64_t p_step, int64_t p_len, const void* q, int64_t q_step, int64_t q_len, int64_t rows) {
  const int64_t p0 = (int64_t)reinterpret_cast<uintptr_t>(p), q0 = (int64_t)reinterpret_cast<uintptr_t>(q);
  const int64_t last = rows - 1;
  if (p_len <= 0 || q_len <= 0) return false;
  if (q0 + last * q_step + q_len <= p0 || p0 + last * p_step + p_len <= q0) return false;
  if (rows == 1 || p_step < p_len || q_step < q_len) return true;
  if (p_step == q_step) {
    // Row j of q begins `in` bytes into the stretch of row j + by of p.
    const int64_t d = q0 - p0, by = d >= 0 ? d / p_step : -((p_step - 1 - d) / p_step), in = d - by * p_step;
    auto both = [&](int64_t shift) { return shift < rows && -shift < rows; };
    return (in < p_len && both(by)) || (in + q_len > p_step && both(by + 1));
  }
  for (int64_t i = 0; i < rows; ++i) {          // the last row of q that begins before the end of p's row i
    const int64_t a = p0 + i * p_step, b = a + p_len;
    if (b <= q0) continue;
    const int64_t j = (b - 1 - q0) / q_step;
    if (q0 + (j < last ? j : last) * q_step + q_len > a) return true;
  }
  return false;
}
// An operand that an output may replace, element by element: it is the output, or apart from it.
inline bool in_place_or_apart(const void* p, int64_t ldp, const void* out, int64_t ldo, int64_t rows, int64_t cols, int64_t e) {
  return (p == out && (ldp == ldo || rows == 1)) || !rows_meet(p, ldp * e, cols * e, out, ldo * e, cols * e, rows);
}

// Whether every row of a (base, stride in elements) matrix starts on a 16-byte boundary.
inline bool rows_16b(const void* p, int64_t ld, int elem_bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * elem_bytes)) & 15) == 0;
}

}  // namespace int8op
