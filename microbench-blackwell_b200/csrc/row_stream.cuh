// row_stream.cuh -- kernels that go through the rows of matrices, a group of threads to a row, with the coming rows
// on their way: copies ahead into shared memory, and the shape of such a launch.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <utility>

#include "row_vec.cuh"
#include "sm100_ptx.cuh"

namespace rowstream {

using rowvec::kUnit;
using rowvec::Unit;

constexpr int kMaxThreads = 512;           // of a group
constexpr int kMaxStages = 4;
constexpr int kSmemLimit = 224 * 1024;     // dynamic shared memory of a block, and of an SM's blocks together

// ----------------------------------------------------------------- rows in flight
// A group of blockDim.x threads (whole warps) takes rows of its own, blockDim.y groups to a block.  A warp copies the
// stretches of the coming rows that its lanes' units make up, 32 units each, into a place of its own in shared memory
// (cp.async: no barrier of the block is needed and no registers are held), one or more rows ahead: the bytes on their way
// are what keeps HBM busy while the group goes through a row's sums.  Lanes copy neighbouring 16-byte chunks (whole
// sectors) and read those of their own unit, so a warp's lanes wait for one another before they read, and before the
// place is copied to again.  Chunk c lies at c ^ (c / 8 mod E): lanes that read E chunks each then meet all banks.
// A stretch off 16-byte boundaries takes one chunk more, and is shifted when it is read.  Every chunk holds
// a byte of the row, so that no copy leaves the 16 bytes around one.
// FULL: all rows start on 16-byte boundaries and every lane's units lie in the row.
// n: elements of the row from the stretch's first on.
template <typename T, bool FULL>
__device__ __forceinline__ void issue_stretch(uint32_t place, const uint8_t* p, int n) {
  constexpr int E = (int)sizeof(T);
  const int lane = (int)(threadIdx.x & 31u);
  const int off = FULL ? 0 : (int)(reinterpret_cast<uintptr_t>(p) & 15u);
  const uint32_t dst = place + 16u * (uint32_t)(lane ^ ((lane >> 3) & (E - 1)));
  const uint8_t* const src = p - off + 16 * lane;
  if (FULL || n >= 32 * kUnit) {
#pragma unroll
    for (int j = 0; j < E; ++j) sm100::cp_async_16(dst + 512u * j, src + 512 * j, 16u);
    if (!FULL && off && lane == 0) sm100::cp_async_16(dst + 512u * E, src + 512 * E, 16u);
  } else if (n > 0) {
    const int chunks = (off + n * E + 15) / 16;
#pragma unroll
    for (int j = 0; j <= E; ++j)
      if (32 * j + lane < chunks) sm100::cp_async_16(dst + 512u * j, src + 512 * j, 16u);
  }
}
// A lane's unit; off: the stretch's offset from a 16-byte boundary, n: elements of the row from the unit's first on.
template <typename T, bool FULL>
__device__ __forceinline__ Unit<T> take_unit(uint32_t place, uint32_t off, int n) {
  constexpr int W = Unit<T>::W, E = (int)sizeof(T);
  Unit<T> u;
  if (!FULL && n <= 0) {
    u.clear();
    return u;
  }
  const int first = E * (int)(threadIdx.x & 31u);
  auto chunk = [&](int j, uint32_t* w) {
    const int c = first + j;
    const uint4 v = sm100::ld_shared_v4(place + 16u * (uint32_t)(c ^ ((c >> 3) & (E - 1))));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  };
  if (FULL || off == 0) {
#pragma unroll
    for (int j = 0; j < E; ++j) chunk(j, u.w + 4 * j);
  } else {
    uint32_t w[W + 4];
#pragma unroll
    for (int j = 0; j <= E; ++j) chunk(j, w + 4 * j);
    rowvec::shift_words<W>(w, off);
#pragma unroll
    for (int j = 0; j < W; ++j) u.w[j] = w[j];
  }
  if (!FULL && n < kUnit) rowvec::clip(u, n * E);
  return u;
}
template <typename T, bool FULL>
__device__ __forceinline__ void put_unit(uint8_t* p, const Unit<T>& u, int n) {
  if constexpr (FULL) rowvec::store_aligned<T>(p, u, kUnit);
  else rowvec::store_unit<T>(reinterpret_cast<T*>(p), u, n);
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the newest n groups of this thread's copies have landed.
__device__ __forceinline__ void wait_copies(int n) {
  switch (n) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
  }
}

__device__ __forceinline__ void group_sync() {
  if (blockDim.x == 32) __syncwarp();
  else sm100::named_bar_sync(1 + threadIdx.y, blockDim.x);
}

// Row `row` of a matrix.  (Opaque: the compiler would otherwise carry a running pointer for every chunk of every unit.)
template <typename P>
__device__ __forceinline__ P* row_of(P* base, int64_t row, int64_t ld) {
  P* r = base + row * ld;
  asm volatile("" : "+l"(r));
  return r;
}
// A condition that is the same for all rows, hidden: the compiler would otherwise make a copy of the loop for each case.
__device__ __forceinline__ bool each_row(bool c) {
  int v = c;
  asm volatile("" : "+r"(v));
  return v != 0;
}
// Makes the compiler unpack a unit again instead of holding its elements in registers over a barrier.
template <typename T>
__device__ __forceinline__ void forget(Unit<T>& u) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < Unit<T>::W; ++j) asm volatile("" : "+r"(u.w[j]));
  }
}

// ----------------------------------------------------------------- host
// Threads of a row, rows of a block and blocks, all resident at once.
struct Shape {
  int tx, ty, blocks, stages;
  size_t smem;
};
// `bytes`: shared memory of a warp and row; `most_threads` of a block; `fixed`: shared memory of a block beside the rows'.
inline Shape shape_of(int64_t rows, int units, int per_thread, int bytes, int most_threads = kMaxThreads, int fixed = 0) {
  Shape s;
  s.tx = ((units + per_thread - 1) / per_thread + 31) / 32 * 32;
  const int warps = s.tx / 32;
  const int room = kSmemLimit - fixed;
  int64_t ty = most_threads / s.tx;
  const int64_t spread = (rows + 147) / 148;       // rows over all SMs before more of them in a block
  if (ty > spread) ty = spread;
  if (ty > room / (bytes * warps)) ty = room / (bytes * warps);
  if (ty > (s.tx == 32 ? 32 : 15)) ty = s.tx == 32 ? 32 : 15;       // named barriers
  s.ty = (int)(ty < 1 ? 1 : ty);
  const int threads = s.tx * s.ty, row_bytes = bytes * warps * s.ty;
  int resident = fixed ? 1 : most_threads / threads;
  if (resident > room / row_bytes) resident = room / row_bytes;      // at least one row ahead
  if (resident < 1) resident = 1;
  const int64_t blocks = (rows + s.ty - 1) / s.ty, most = 148 * resident;
  s.blocks = (int)(blocks < most ? blocks : most);
  s.stages = room / resident / row_bytes;
  if (s.stages > kMaxStages) s.stages = kMaxStages;
  const int64_t each = (rows + (int64_t)s.blocks * s.ty - 1) / ((int64_t)s.blocks * s.ty);
  if (s.stages > each) s.stages = (int)each;
  s.smem = (size_t)s.stages * row_bytes;
  return s;
}

// A stretch in shared memory.
inline uint32_t place_bytes(int e, bool wide) { return (uint32_t)(32 * e + (wide ? 0 : 1)) * 16u; }
// `units` of a row among threads of `per_thread` each: every one is there.
inline bool all_full(int units, int cols, int per_thread) { return units % (32 * per_thread) == 0 && cols == units * kUnit; }
// Whether the rows of all matrices start on 16-byte boundaries (strides in bytes; an absent one does not count).
inline bool all_wide(std::initializer_list<std::pair<const void*, int64_t>> matrices) {
  uintptr_t bits = 0;
  for (const auto& m : matrices)
    if (m.first) bits |= reinterpret_cast<uintptr_t>(m.first) | (uintptr_t)m.second;
  return (bits & 15) == 0;
}

}  // namespace rowstream
