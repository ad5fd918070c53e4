// int8_gemv.cuh -- the few-token form of the int8 product (int8_gemv.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "int8_common.cuh"

namespace int8op {

constexpr int kGemvTokens = 4;          // most tokens of the few-token form
constexpr int kTypeInt8 = -1;           // GemvParams.x_type of tokens that are quantised already

struct GemvParams {
  const void* x; int64_t ldx;           // tokens; elements
  const int8_t* b; int64_t ldb;
  void* d; int64_t ldd;
  const void* c; int64_t ldc;
  const float* sa;                      // scales of int8 tokens (NULL = 1)
  const float* sb;
  const void* bias;
  int32_t x_type, d_type, bias_type;
  int32_t m, n, k;
  int32_t wide;                         // rows of floating x start on 16-byte boundaries
  int32_t depth;                        // ring slots of a warp, set by gemv_launch
  int32_t* status;
  uint64_t timeout_ns;
  Drop drop;
};

// Whether the tokens fit in a block's shared memory.
bool gemv_fits(int64_t m, int64_t n, int64_t k, int num_sms);
cudaError_t gemv_launch(const GemvParams& p, int num_sms, cudaStream_t st);

}  // namespace int8op
