// counter_rng.cuh -- the library's counter-based generator: every draw is a
// pure function of (seed, stream, index), splitmix64 over a per-stream key.
#pragma once
#include <cstdint>

namespace counter_rng {

constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ULL;

__host__ __device__ __forceinline__ uint64_t mix64(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
  return z ^ (z >> 31);
}
__host__ __device__ __forceinline__ uint64_t stream_key(uint64_t seed, uint64_t stream) {
  return mix64(seed + mix64(stream + kGolden));
}
// The 64 bits of draw `index`.
__host__ __device__ __forceinline__ uint64_t draw(uint64_t key, uint64_t index) {
  return mix64(key + (index + 1) * kGolden);
}

}  // namespace counter_rng
