// fp4_common.cuh -- 4-bit floating operands (e2m1 values, a scale for each block of 16 or 32 elements, a
// scale for each row): the rounding, shared by the quantiser, the few-token product and the norm that
// writes such an operand, and where the block scales lie.
//
//   g = 2^(floor(log2 max|x|) - 10), at least 2^-126        row scale; y = x / g is below 2048
//   s = the least e4m3 number (blocks of 16) or power of two of at least 2^-126 (blocks of 32) with 6 s >= max|y|
//   q = y / s rounded to e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6), ties to the even code
//
// The row scale is a power of two, so y is exact, rows do not depend on one another, and the largest block
// scale is in [171, 342) of e4m3's 448: blocks keep three bits of scale down to 2^-14 of the row's largest.
#pragma once
#include <cstdint>

#include "int8_common.cuh"

namespace fp4op {

constexpr float kSixth = 0.16666667f;

// K elements of one 128-byte row of the product's operand, and block scales that are stored for them.
constexpr int kAtomK = 256;
__host__ __device__ constexpr bool block_ok(int block) { return block == 16 || block == 32; }
// Tiles of 128 rows x 4 scales along a row: whole atoms of K.
__host__ __device__ constexpr int64_t scale_tiles(int64_t cols, int block) {
  return (cols + kAtomK - 1) / kAtomK * (kAtomK / 4 / block);
}
// Byte of the scale (row, block column).
__host__ __device__ constexpr int64_t scale_at(int64_t row, int64_t col, int64_t tiles) {
  return ((row >> 7) * tiles + (col >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (col & 3);
}

struct RowScale {
  float up;      // 1 / g
  float scale;   // g, or the NaN or Inf of the row, whose elements then count as zeros
  __device__ __forceinline__ bool lost() const { return (__float_as_uint(scale) & 0x7F800000u) == 0x7F800000u; }
  // g is so far from 1 that it has to be applied to the elements (which is exact) before anything else: the
  // scales of their blocks in x's own unit might leave fp32's range.
  __device__ __forceinline__ bool far() const { return !(scale > 0x1p-100f && scale < 0x1p100f); }
};
// `bits`: the largest |x| of the row as fp32 bits (integer maximum, so NaN > Inf > finite).
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale s;
  if (bits >= 0x7F800000u) {
    s.up = 1.f;
    s.scale = __uint_as_float(bits);
    return s;
  }
  const uint32_t e = max(bits >> 23, 11u);
  s.up = __uint_as_float((264u - e) << 23);
  s.scale = __uint_as_float((e - 10u) << 23);
  return s;
}

__device__ __forceinline__ float decode_e4m3(uint32_t code) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(code));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}
__device__ __forceinline__ float decode_e8m0(uint32_t code) {
  return code == 0u ? 0x1p-127f : (code == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(code << 23));
}

struct BlockScale {
  uint32_t code;
  float s, r;      // the scale and 1 / s rounded to nearest (0 for s = 0)
};
// From the largest |y| of a block, finite and below 2048.
//  e4m3: top / 6 rounded up to four significant bits (from 2^-6 on; in steps of 2^-9 below), and one step more where 6 times that
//    is still below top.  (fp32's 1/6 times 6 s rounds back to s, so a top that is exactly 6 s stays at s.)  1 / s: one Newton
//    step from the approximation is 2^-46 off, and no 8 / (8 + m) is that near to the middle of two fp32 numbers.
//  e8m0: 6 * 2^k >= 2^e m with k = e - 2 for m <= 3/2, else e - 1.
template <int BLOCK>
__device__ __forceinline__ BlockScale block_scale(float top) {
  BlockScale b;
  if constexpr (BLOCK == 16) {
    const float t = top * kSixth;
    if (t >= 0x1p-6f) {
      uint32_t u = (__float_as_uint(t) + 0xFFFFFu) & 0xFFF00000u;
      if (6.f * __uint_as_float(u) < top) u += 0x100000u;
      b.code = (u >> 20) - 8u * (127u - 7u);
      b.s = __uint_as_float(u);
    } else {
      b.code = __float2uint_ru(t * 512.f);
      if ((float)b.code * (6.f / 512.f) < top) ++b.code;
      b.s = (float)b.code * 0x1p-9f;
    }
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b.s));
    b.r = b.s > 0.f ? fmaf(fmaf(-b.s, r, 1.f), r, r) : 0.f;
  } else {
    const uint32_t u = __float_as_uint(top);
    const int k = (int)(u >> 23) - 2 + ((u & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    b.code = (uint32_t)max(k, 1);
    b.s = __uint_as_float(b.code << 23);
    b.r = __uint_as_float((254u - b.code) << 23);
  }
  return b;
}

// Eight values to a word, the first in the low four bits; |z| <= 6.
__device__ __forceinline__ uint32_t pack8(const float (&z)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w) : "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]), "f"(z[4]), "f"(z[5]), "f"(z[6]), "f"(z[7]));
  return w;
}

// Codes of 8 elements x = g y of a block.  The quotient y / s has to be decided exactly at the seven borders
// between codes, where bf16 blocks lie often: one correction of x (r / g) gives it rounded to nearest (r being 1 / s
// rounded to nearest, and g a power of two), and a quotient that is not a border, with s of four bits and y of 24, does
// not round to one.  Division by powers of two is exact as it is (in two steps: together they might leave fp32's range).
template <int BLOCK>
__device__ __forceinline__ uint32_t round8(const float* x, const BlockScale& b, float up, float g) {
  using int8op::F2;
  float z[8];
  const F2 r(b.r * up, b.r * up), ns(-b.s * g, -b.s * g), r1(b.r, b.r), u(up, up);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const F2 v(x[j], x[j + 1]);
    F2 t;
    if constexpr (BLOCK == 16) {
      t = int8op::mul2(v, r);
      t = int8op::fma2(int8op::fma2(ns, t, v), r, t);
    } else {
      t = int8op::mul2(int8op::mul2(v, u), r1);
    }
    t.get(z[j], z[j + 1]);
  }
  return pack8(z);
}

// Elements of a row that is far from 1, and the largest of them, times 1 / g; zeros for a row that is lost.
__device__ __forceinline__ void bring_near(float (&x)[16], float& top, const RowScale& s) {
  const bool lost = s.lost();
  top = lost ? 0.f : top * s.up;
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = lost ? 0.f : x[j] * s.up;
}

// The 16 elements of a thread's unit (a warp's lanes hold consecutive units of a row; all of them call) and the largest
// magnitude among them: codes in two words, and this block's scale code.  Blocks of 32 are two lanes'.
template <int BLOCK>
__device__ __forceinline__ uint32_t quantize_unit(const float (&x)[16], float top, float up, float g, uint32_t (&q)[2]) {
  if constexpr (BLOCK == 32) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  const BlockScale b = block_scale<BLOCK>(top * up);
  q[0] = round8<BLOCK>(x, b, up, g);
  q[1] = round8<BLOCK>(x + 8, b, up, g);
  return b.code;
}

// Stores the scale codes of a warp's units: four blocks to a word.  `unit`: this lane's in the row, a multiple of the
// lane modulo 32; `live`: the row and unit exist (units come in whole atoms of K, so groups of four blocks are alike).
template <int BLOCK>
__device__ __forceinline__ void store_scale_codes(uint8_t* scales, int64_t row, int64_t tiles, int unit, uint32_t code, bool live) {
  constexpr int STEP = BLOCK / 16;                       // lanes of a block
  const int lane = (int)(threadIdx.x & 31u);
  uint32_t v = code << (8 * ((lane / STEP) & 3));
  v |= __shfl_xor_sync(0xFFFFFFFFu, v, STEP);
  v |= __shfl_xor_sync(0xFFFFFFFFu, v, 2 * STEP);
  if (live && (lane & (4 * STEP - 1)) == 0) *reinterpret_cast<uint32_t*>(scales + scale_at(row, unit / STEP, tiles)) = v;
}

// The 8 bytes of a unit's values; `n`: elements of the unit in the row.
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&q)[2], int n) {
  if (n >= 16) {
    *reinterpret_cast<uint2*>(p) = make_uint2(q[0], q[1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (2 * j < n) {
        uint32_t b = (q[j / 4] >> (8 * (j & 3))) & 0xFFu;
        if (2 * j + 1 >= n) b &= 0xFu;
        p[j] = (uint8_t)b;
      }
  }
}

}  // namespace fp4op
