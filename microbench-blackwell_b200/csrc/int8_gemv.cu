// int8_gemv.cu -- the int8 linear layer for a few tokens: quantisation, product
// and epilogue in one launch.
//
// Bound by the bytes of the weights.  One block per SM owns a contiguous range
// of channels; its warps split the (channel pair, 2048-byte K chunk) units of
// that range evenly, so all SMs and warps finish together.  Each warp streams its
// own units through a private ring in shared memory (bulk copies that the
// warp itself refills, no producer), 192 KB in flight per SM.  The first of them
// are issued before the tokens are touched: every block then finds the tokens'
// maxima, quantises them into its shared memory (they are a few KB, read
// through L2) and multiplies with dp4a.  The int32 sums are exact, so the result
// has the bits of the tensor-core kernel.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "gemm_sm100a.h"
#include "int8_common.cuh"
#include "int8_gemv.cuh"
#include "sm100_ptx.cuh"

using namespace int8op;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kLoads = 4;                       // 512-byte rows of a channel's chunk
constexpr int kChunk = kLoads * 512;            // K bytes of one unit
constexpr int kSlot = 2 * kChunk;               // one unit: two channels
constexpr int kMaxDepth = 3;                    // units in flight per warp
constexpr int kMaxSmem = 224 * 1024;

// Tokens of X quantised into xq[t][kpad] (zero beyond k) with scale[t]; whole block.
template <typename X, int MT>
__device__ __forceinline__ void stage_tokens(const GemvParams& p, int8_t* xq, float* scale, uint32_t* top, int kpad) {
  if constexpr (sizeof(X) == 1) {
    for (int i = threadIdx.x; i < MT * (kpad / 16); i += kThreads) {
      const int t = i / (kpad / 16), k = (i - t * (kpad / 16)) * 16;
      int4 v = make_int4(0, 0, 0, 0);
      if (t < p.m) {
        const int8_t* src = static_cast<const int8_t*>(p.x) + t * p.ldx + k;
        if (k + 16 <= p.k) {
          v = *reinterpret_cast<const int4*>(src);
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (k + j < p.k) w[j / 4] |= (uint32_t)(uint8_t)src[j] << (8 * (j & 3));
          v = make_int4((int)w[0], (int)w[1], (int)w[2], (int)w[3]);
        }
      }
      *reinterpret_cast<int4*>(xq + t * kpad + k) = v;
    }
    if (threadIdx.x < MT) scale[threadIdx.x] = p.sa && threadIdx.x < p.m ? p.sa[threadIdx.x] : 1.f;
    __syncthreads();
  } else {
    constexpr int V = Vec<X>::N;
    constexpr int HOLD = 4;                     // vectors a thread keeps between the two passes
    const int nvec = kpad / V, total = p.m * nvec;
    Vec<X> v[HOLD];
    auto load = [&](int i) {
      const int t = i / nvec, e = (i - t * nvec) * V;
      return load_vec<X>(static_cast<const X*>(p.x) + t * p.ldx + e, p.k - e, p.wide);
    };
    auto magnitude = [&](const Vec<X>& a) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(X) == 4) m = max(m, a.w[j] & 0x7FFFFFFFu);
        else m = __vmaxu2(m, a.w[j] & 0x7FFF7FFFu);
      }
      if constexpr (sizeof(X) == 2) m = abs_bits_to_f32<X>(max(m & 0xFFFFu, m >> 16));
      return m;
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
      const int i = h * kThreads + (int)threadIdx.x;
      if (i < total) v[h] = load(i);
    }
    if (threadIdx.x < MT) top[threadIdx.x] = 0u;
    __syncthreads();
    // One shared atomic per warp and row: a warp's 32 vectors are mostly of one row.
    auto join = [&](int i, uint32_t m) {   // whole warp
      const int t = MT == 1 ? 0 : min(i, total - 1) / nvec;
      if (MT == 1 || __all_sync(0xFFFFFFFFu, t == __shfl_sync(0xFFFFFFFFu, t, 0))) {
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((threadIdx.x & 31) == 0) atomicMax(&top[t], m);
      } else {
        atomicMax(&top[t], m);
      }
    };
    const int warp0 = (int)(threadIdx.x & ~31u);
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
      const int i = h * kThreads + (int)threadIdx.x;
      if (h * kThreads + warp0 < total) join(i, i < total ? magnitude(v[h]) : 0u);
    }
    for (int i0 = HOLD * kThreads + warp0; i0 < total; i0 += kThreads) {
      const int i = i0 + (int)(threadIdx.x & 31);
      join(i, i < total ? magnitude(load(i)) : 0u);
    }
    __syncthreads();
    auto write = [&](int i, const Vec<X>& a) {
      const int t = i / nvec, e = (i - t * nvec) * V;
      const RowScale s = row_scale(top[t]);
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        uint32_t w = pack4(quantize_one<X>(a.get(4 * j), s), quantize_one<X>(a.get(4 * j + 1), s),
                           quantize_one<X>(a.get(4 * j + 2), s), quantize_one<X>(a.get(4 * j + 3), s));
        if (s.c == 0.f) w = 0u;
        *reinterpret_cast<uint32_t*>(xq + t * kpad + e + 4 * j) = w;
      }
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
      const int i = h * kThreads + (int)threadIdx.x;
      if (i < total) write(i, v[h]);
    }
    for (int i = HOLD * kThreads + threadIdx.x; i < total; i += kThreads) write(i, load(i));
    for (int i = total * V + 4 * threadIdx.x; i < MT * kpad; i += 4 * kThreads) *reinterpret_cast<uint32_t*>(xq + i) = 0u;
    if (threadIdx.x < p.m) scale[threadIdx.x] = row_scale(top[threadIdx.x]).scale;
    __syncthreads();
  }
}

// Wait for a ring slot, within the time budget.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t phase, const GemvParams& p) {
  const uint64_t t0 = sm100::globaltimer_ns();
  while (!sm100::mbar_try_wait(bar, phase)) {
    if (sm100::globaltimer_ns() - t0 > p.timeout_ns) {
      if (p.status) atomicCAS(p.status, 0, (int32_t)(0x3u | (1u << 8) | ((blockIdx.x & 0x7FFu) << 20)));
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t phase, const GemvParams& p) {
  const bool ok = sm100::mbar_try_wait(bar, phase) || wait_slow(bar, phase, p);
  return __all_sync(0xFFFFFFFFu, ok);
}

// 16 bytes of a row that ends after `n` of them.
__device__ __forceinline__ int4 load_tail(const int8_t* p, int n) {
  uint32_t t[4] = {0, 0, 0, 0};
  for (int j = 0; j < n; ++j) t[j / 4] |= (uint32_t)(uint8_t)p[j] << (8 * (j & 3));
  return make_int4((int)t[0], (int)t[1], (int)t[2], (int)t[3]);
}

template <typename X, int MT>
__global__ void __launch_bounds__(kThreads, 1) int8_gemv_kernel(const __grid_constant__ GemvParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float scale[MT];
  __shared__ uint32_t top[MT];
  __shared__ __align__(8) uint64_t full[kWarps][kMaxDepth];
  const int kpad = (p.k + 15) & ~15;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // [ring][tokens: MT x kpad][sums: channels of this block x MT]
  const uint32_t ring = sm100::smem_u32(smem) + (uint32_t)(warp * p.depth * kSlot);
  int8_t* const xq = reinterpret_cast<int8_t*>(smem + (size_t)kWarps * p.depth * kSlot);
  int32_t* const sums = reinterpret_cast<int32_t*>(xq + (size_t)MT * kpad);
  const uint32_t bar = sm100::smem_u32(&full[warp][0]);

  const int pairs = (p.n + 1) / 2;
  const int pair0 = (int)((int64_t)blockIdx.x * pairs / gridDim.x);
  const int pair1 = (int)((int64_t)(blockIdx.x + 1) * pairs / gridDim.x);
  const int chunks = (kpad + kChunk - 1) / kChunk;
  const int units = (pair1 - pair0) * chunks;
  const int u_begin = (int)((int64_t)warp * units / kWarps);
  const int u_end = (int)((int64_t)(warp + 1) * units / kWarps);
  const uint64_t policy = sm100::policy_evict_normal();
  const bool ragged = (p.k & 15) != 0;          // the matrix may end inside the last 16 bytes of its last row

  auto issue = [&](int unit, int slot) {        // lane 0
    const int pr = unit / chunks, k0 = (unit - pr * chunks) * kChunk;
    const int ch = 2 * (pair0 + pr);
    const int whole = min(kChunk, kpad - k0);
    int b0 = whole, b1 = ch + 1 < p.n ? whole : 0;
    if (ragged && whole == kpad - k0) {
      if (ch + 1 == p.n) b0 -= 16;
      if (ch + 2 == p.n) b1 -= 16;
    }
    const uint32_t dst = ring + (uint32_t)(slot * kSlot);
    const int8_t* src = p.b + (int64_t)ch * p.ldb + k0;
    sm100::mbar_arrive_expect_tx(bar + 8u * slot, (uint32_t)(b0 + b1));
    if (b0 > 0) sm100::bulk_load(dst, src, (uint32_t)b0, bar + 8u * slot, policy);
    if (b1 > 0) sm100::bulk_load(dst + kChunk, src + p.ldb, (uint32_t)b1, bar + 8u * slot, policy);
  };
  if (lane == 0) {
    for (int s = 0; s < p.depth; ++s) sm100::mbar_init(bar + 8u * s, 1);
    sm100::fence_mbar_init();
  }
  __syncwarp();
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  if (lane == 0)
    for (int s = 0; s < p.depth && u_begin + s < u_end; ++s) issue(u_begin + s, s);

  for (int i = threadIdx.x; i < 2 * (pair1 - pair0) * MT; i += kThreads) sums[i] = 0;
  stage_tokens<X, MT>(p, xq, scale, top, kpad);

  int32_t acc[2][MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[0][t] = acc[1][t] = 0;
  int slot = 0;
  uint32_t phase = 0;
  for (int u = u_begin; u < u_end; ++u) {
    if (!wait_full(bar + 8u * slot, phase, p)) {
      // Give the copies in flight a bounded time to land before the block may exit.
      for (int r = 0; r < p.depth && u + r < u_end; ++r) {
        const int s = slot + r < p.depth ? slot + r : slot + r - p.depth;
        const uint64_t t0 = sm100::globaltimer_ns();
        while (!sm100::mbar_try_wait(bar + 8u * s, slot + r < p.depth ? phase : phase ^ 1u) &&
               sm100::globaltimer_ns() - t0 < 100000000ull) {}
      }
      break;
    }
    const int pr = u / chunks;
    const int kc = (u - pr * chunks) * kChunk, ch = 2 * (pair0 + pr);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int o = i * 512 + lane * 16, k = kc + o;
      if (k < kpad) {
        int4 w[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint4 v = sm100::ld_shared_v4(ring + (uint32_t)(slot * kSlot + c * kChunk + o));
          w[c] = make_int4((int)v.x, (int)v.y, (int)v.z, (int)v.w);
          if (ragged && k + 16 > p.k && ch + c + 1 >= p.n) {
            w[c] = ch + c < p.n ? load_tail(p.b + (int64_t)(ch + c) * p.ldb + k, p.k - k) : make_int4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int4 x = *reinterpret_cast<const int4*>(xq + t * kpad + k);
#pragma unroll
          for (int c = 0; c < 2; ++c)
            acc[c][t] = __dp4a(w[c].x, x.x, __dp4a(w[c].y, x.y, __dp4a(w[c].z, x.z, __dp4a(w[c].w, x.w, acc[c][t]))));
        }
      }
    }
    __syncwarp();
    if (lane == 0 && u + p.depth < u_end) issue(u + p.depth, slot);
    if (++slot == p.depth) { slot = 0; phase ^= 1u; }
    if (u + 1 == u_end || (u + 1) / chunks != pr) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int32_t s = __reduce_add_sync(0xFFFFFFFFu, acc[c][t]);
          if (lane == 0) atomicAdd(&sums[(2 * pr + c) * MT + t], s);
          acc[c][t] = 0;
        }
    }
  }
  __syncthreads();
  const int nch = min(2 * (pair1 - pair0), p.n - 2 * pair0);
  const uint64_t key = p.drop.on ? drop_key(p.drop) : 0;
  for (int i = threadIdx.x; i < nch * MT; i += kThreads) {
    const int t = i / nch, c = i - t * nch;
    if (t >= p.m) continue;
    const int64_t ch = 2 * pair0 + c;
    float v = finish(sums[c * MT + t], scale[t], p.sb ? p.sb[ch] : 1.f, p.bias ? load_as_f32(p.bias, p.bias_type, ch) : 0.f);
    if (p.drop.on) v = drop_keeps(key, p.drop.threshold, drop_index(p.drop, t, ch)) ? v * p.drop.grow : 0.f;
    if (p.c) v += load_as_f32(p.c, p.d_type, t * p.ldc + ch);
    store_as(p.d, p.d_type, t * p.ldd + ch, v);
  }
}

int grid_of(int64_t n, int num_sms) {
  const int64_t pairs = (n + 1) / 2;
  return (int)(pairs < num_sms ? pairs : num_sms);
}
// Tokens, then one sum per token and channel of the largest block.
int64_t fixed_smem(int mt, int64_t n, int64_t k, int num_sms) {
  const int grid = grid_of(n, num_sms);
  return (int64_t)mt * ((k + 15) & ~15) + ((n + 1) / 2 + grid - 1) / grid * 2 * mt * 4;
}
int depth_of(int mt, int64_t n, int64_t k, int num_sms) {
  const int64_t d = (kMaxSmem - fixed_smem(mt, n, k, num_sms)) / (kWarps * kSlot);
  return (int)(d > kMaxDepth ? kMaxDepth : d);
}

template <typename X, int MT>
cudaError_t run(GemvParams p, int num_sms, cudaStream_t st) {
  p.depth = depth_of(MT, p.n, p.k, num_sms);
  const size_t smem = (size_t)(kWarps * p.depth * kSlot + fixed_smem(MT, p.n, p.k, num_sms));
  const cudaError_t e = cudaFuncSetAttribute(int8_gemv_kernel<X, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) return e;
  return launch_overlapped(int8_gemv_kernel<X, MT>, dim3(grid_of(p.n, num_sms)), dim3(kThreads), smem, 1, st, p);
}

template <typename X>
cudaError_t by_tokens(const GemvParams& p, int num_sms, cudaStream_t st) {
  if (p.m == 1) return run<X, 1>(p, num_sms, st);
  if (p.m == 2) return run<X, 2>(p, num_sms, st);
  return run<X, 4>(p, num_sms, st);
}

}  // namespace

namespace int8op {

bool gemv_fits(int64_t m, int64_t n, int64_t k, int num_sms) {
  if (m < 1 || m > kGemvTokens || n < 1) return false;
  return depth_of((int)(m == 3 ? 4 : m), n, k, num_sms) >= 1;
}

cudaError_t gemv_launch(const GemvParams& p, int num_sms, cudaStream_t st) {
  switch (p.x_type) {
    case GEMM_TYPE_BF16: return by_tokens<__nv_bfloat16>(p, num_sms, st);
    case GEMM_TYPE_FP16: return by_tokens<__half>(p, num_sms, st);
    case GEMM_TYPE_FP32: return by_tokens<float>(p, num_sms, st);
    default: return by_tokens<int8_t>(p, num_sms, st);
  }
}

}  // namespace int8op
