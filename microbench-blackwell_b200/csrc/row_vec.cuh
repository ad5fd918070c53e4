// row_vec.cuh -- rows of a matrix in units of 16 consecutive elements per thread, at any alignment of
// the rows.
//
// Contiguous tensors whose rows have an odd length start most rows off 16-byte boundaries.  Element by element
// such a row takes 16 loads per unit; here it takes the 16-byte blocks that the unit touches and a
// shift by the row's misalignment, the same for all of its units.  A block is read whole where
// any byte of it belongs to the row: it lies in the same 16 bytes of memory as that one, so the read
// stays in range of the allocation, and what is not the row's is dropped.
#pragma once
#include <cstdint>

#include "int8_common.cuh"

namespace rowvec {

using namespace int8op;

constexpr int kUnit = 16;      // elements of a unit

// Words [0, N) of `w` become those `bytes` (0..14, even) further on; w has N + 4 words.
template <int N>
__device__ __forceinline__ void shift_words(uint32_t (&w)[N + 4], uint32_t bytes) {
  if (bytes & 8u) {
#pragma unroll
    for (int j = 0; j < N + 2; ++j) w[j] = w[j + 2];
  }
  if (bytes & 4u) {
#pragma unroll
    for (int j = 0; j < N + 1; ++j) w[j] = w[j + 1];
  }
  if (bytes & 2u) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
  }
}

// A unit of T as packed words.
template <typename T>
struct Unit {
  static constexpr int W = kUnit * (int)sizeof(T) / 4;
  uint32_t w[W];
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
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = 0u;
  }
};

// Largest |x| of a unit as fp32 bits (integer maximum, so NaN > Inf > finite).
template <typename T>
__device__ __forceinline__ uint32_t magnitude(const Unit<T>& u) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < Unit<T>::W; ++j) {
    if constexpr (sizeof(T) == 4) m = max(m, u.w[j] & 0x7FFFFFFFu);
    else m = __vmaxu2(m, u.w[j] & 0x7FFF7FFFu);
  }
  if constexpr (sizeof(T) == 2) m = abs_bits_to_f32<T>(max(m & 0xFFFFu, m >> 16));
  return m;
}
// Zeros beyond the first `bytes` of a unit.
template <typename T>
__device__ __forceinline__ void clip(Unit<T>& u, int bytes) {
  if (bytes < 4 * Unit<T>::W) {
#pragma unroll
    for (int j = 0; j < Unit<T>::W; ++j) {
      const int left = bytes - 4 * j;
      if (left < 4) u.w[j] = left == 2 ? u.w[j] & 0xFFFFu : 0u;
    }
  }
}

// 32 bytes at once: a thread's 16-bit unit, or half of an fp32 one.  (Lanes 32 bytes apart that move 16 at a time ask
// for every sector twice: residual_norm of 16384 x 8192 bf16 took 292 us that way, 199 with whole sectors.)
template <bool STREAM>
__device__ __forceinline__ void load32(uint32_t* w, const uint8_t* p) {
  if constexpr (STREAM)
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
  else
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store32(uint8_t* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

enum Cache { kStream, kKeep };   // read once, or again by other rows

template <Cache C>
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 v;
  if constexpr (C == kStream)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  else
    v = *reinterpret_cast<const uint4*>(p);
  return v;
}

// Elements [0, n) of a unit at p (n <= 0: none; the rest reads as 0).  p is aligned to T.
template <typename T, Cache C = kStream>
__device__ __forceinline__ Unit<T> load_unit(const T* ptr, int n) {
  constexpr int W = Unit<T>::W, B = W / 4;
  const uint8_t* const p = reinterpret_cast<const uint8_t*>(ptr);
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const int bytes = min(n, kUnit) * (int)sizeof(T);
  Unit<T> u;
  if (n >= kUnit && ((uint32_t)reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
#pragma unroll
    for (int j = 0; j < W / 8; ++j) load32<C == kStream>(u.w + 8 * j, p + 32 * j);
    return u;
  }
  if (off == 0) {
#pragma unroll
    for (int j = 0; j < B; ++j) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (16 * j < bytes) v = load16<C>(p + 16 * j);
      u.w[4 * j] = v.x; u.w[4 * j + 1] = v.y; u.w[4 * j + 2] = v.z; u.w[4 * j + 3] = v.w;
    }
  } else {
    uint32_t w[W + 4];
#pragma unroll
    for (int j = 0; j <= B; ++j) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (bytes > 0 && 16 * j - (int)off < bytes) v = load16<C>(p - off + 16 * j);
      w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
    }
    shift_words<W>(w, off);
#pragma unroll
    for (int j = 0; j < W; ++j) u.w[j] = w[j];
  }
  clip(u, bytes);
  return u;
}

// Elements [a, b) of a unit, one by one.
template <typename T>
__device__ __forceinline__ void store_elements(T* p, const Unit<T>& u, int a, int b) {
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    if (i >= a && i < b) {
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[i] = u.w[i];
      else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(i & 1 ? u.w[i / 2] >> 16 : u.w[i / 2] & 0xFFFFu);
    }
}

// Elements [0, n) of a unit at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_aligned(uint8_t* p, const Unit<T>& u, int n) {
  constexpr int W = Unit<T>::W;
  if (n >= kUnit) {
    if (((uint32_t)reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
#pragma unroll
      for (int j = 0; j < W / 8; ++j) store32(p + 32 * j, u.w + 8 * j);
    } else {
#pragma unroll
      for (int j = 0; j < W / 4; ++j) *reinterpret_cast<uint4*>(p + 16 * j) = make_uint4(u.w[4 * j], u.w[4 * j + 1], u.w[4 * j + 2], u.w[4 * j + 3]);
    }
  } else if (n > 0) {
    store_elements<T>(reinterpret_cast<T*>(p), u, 0, n);
  }
}

// Bytes [from, to) of the 16 at q, from words: at most one 16-bit piece at either end, where a 16-bit element ends there.
__device__ __forceinline__ void store_part(uint8_t* q, const uint32_t* w, uint32_t from, uint32_t to) {
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    if (from <= 4 * j && 4 * j + 4 <= to) *reinterpret_cast<uint32_t*>(q + 4 * j) = w[j];
    else if (from <= 4 * j && 4 * j + 2 == to) *reinterpret_cast<uint16_t*>(q + 4 * j) = (uint16_t)w[j];
    else if (from == 4 * j + 2 && 4 * j + 4 <= to) *reinterpret_cast<uint16_t*>(q + 4 * j + 2) = (uint16_t)(w[j] >> 16);
  }
}

// Elements [0, n) of the units of a warp, called by all of its lanes; lane l + 1's unit follows lane l's in the
// row (of other lanes' rows nothing is assumed).  Off 16-byte boundaries a lane also writes the end of the
// unit before it, so that whole blocks are written; only at both ends of the warp's stretch, and at the row's end, parts are.
template <typename T>
__device__ __forceinline__ void store_unit(T* ptr, const Unit<T>& u, int n) {
  constexpr int W = Unit<T>::W, B = W / 4, E = (int)sizeof(T);
  uint8_t* const p = reinterpret_cast<uint8_t*>(ptr);
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  if (off == 0) {      // uniform over the warp
    store_aligned<T>(p, u, n);
    return;
  }
  uint32_t w[W + 4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = __shfl_up_sync(0xFFFFFFFFu, u.w[W - 4 + j], 1);
#pragma unroll
  for (int j = 0; j < W; ++j) w[4 + j] = u.w[j];
  const int head = (16 - (int)off) / E;      // own elements in the block that begins in the unit before
  const int lane = (int)(threadIdx.x & 31u);
  uint8_t* const q = p - off;
  shift_words<W>(w, 16u - off);              // words of the blocks from q
  if (n >= kUnit) {
    if (lane > 0) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    else store_part(q, w, off, 16u);
#pragma unroll
    for (int j = 1; j < B; ++j) *reinterpret_cast<uint4*>(q + 16 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    if (lane == 31 || n - kUnit < head) {    // the next lane has nothing, or not enough, to fill the block with
      uint32_t t[8] = {u.w[W - 4], u.w[W - 3], u.w[W - 2], u.w[W - 1], 0u, 0u, 0u, 0u};
      shift_words<4>(t, 16u - off);
      store_part(q + 16 * B, t, 0u, off);
    }
  } else if (n > 0) {
    int done = 0;
    if (lane > 0 && n >= head) {             // the unit before is full
      *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
      done = head;
    }
    store_elements<T>(ptr, u, done, n);
  }
}

}  // namespace rowvec
