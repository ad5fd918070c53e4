// int8_gemm.cu -- product of int8 operands with one scale per token and channel:
//   D[i][j] = C[i][j] + dropout(sa[i] * sb[j] * sum_k A[i][k] B[j][k] + bias[j])
//
// tcgen05.mma kind::i8 (int32 accumulators in TMEM): the sum is exact, so every
// tiling, split and batch gives the same bits.
//
// Channels (rows of B) lie on the MMA's M side, tokens (rows of A) on its N
// side: an accumulator lane is one channel, a column one token.  The weight
// tile is then always a full 128 rows however few tokens there are, a
// thread keeps its channel's scale and bias in registers, and a warp's 32 lanes
// write 32 consecutive elements of a row of D.
//
// Warp 0 loads 128-byte K atoms by TMA into a ring, warp 1 issues the MMAs,
// warps 2..5 run the epilogue (one TMEM lane quadrant each).
//   whole-K form   persistent CTAs (CTA pairs for large problems), two
//                  accumulators, so a tile's epilogue overlaps the next mainloop.
//   split-K form   for few tiles: the CTAs of a cluster share one tile's K and
//                  add their int32 partial tiles through distributed shared
//                  memory (exact, so the order does not matter); no workspace.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "gemm_sm100a.h"
#include "sm100_ptx.cuh"
#include "bounded_wait.cuh"
#include "device_guard.cuh"
#include "int8_common.cuh"
#include "int8_gemv.cuh"
#include "tensor_map.cuh"

using namespace sm100;
using namespace int8op;

namespace {

constexpr int kThreads = 192;
constexpr int kSmemLimit = 232448;      // 227 KiB of opt-in dynamic shared memory per CTA
constexpr int kBarrierBytes = 1024;
constexpr int kMaxStages = 32;
constexpr int kAtom = 128;              // bytes (= K elements) of one swizzled K atom
constexpr int kChannels = 128;          // channels per CTA
constexpr int kMaxSplit = 8;            // CTAs that may share a tile's K (portable cluster size)

struct Int8Params {
  void* d; int64_t ldd;
  const void* c; int64_t ldc;
  const float* sa;
  const float* sb;
  const void* bias;
  int32_t bias_type;
  int32_t m, n;
  Drop drop;
  int32_t num_cb, num_tb, num_units;    // channel blocks, token blocks, output tiles
  int32_t num_kb;                       // K atoms
  int32_t split;                        // CTAs (a cluster) that share a tile's K; 1 = whole-K form
  int32_t stages;
  uint32_t stage_bytes, a_bytes;        // per CTA: weights, then tokens
  uint32_t bars_offset, stg_offset, sa_offset, stg_bytes;
  int32_t stg_bufs;                     // staging buffers (0 = direct stores)
  int32_t tmem_cols, num_acc;
  int32_t raster;                       // channel blocks per raster group
  uint32_t idesc;
  int32_t* status;
  uint64_t timeout_ns;
  uint32_t flags;
  int32_t weights_ready;                // the kernel before this one does not write the weights
};

// kind::i8: [4,6) D format (2 = S32), [7,10) and [10,13) A and B format (1 = signed
// 8-bit), both K-major, [17,23) N >> 3, [24,29) M >> 4.
__host__ constexpr uint32_t make_idesc(int mma_m, int mma_n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(mma_n >> 3) << 17) | ((uint32_t)(mma_m >> 4) << 24);
}

__device__ __forceinline__ void tile_coords(int u, const Int8Params& p, int& cb, int& tb) {
  const int per_group = p.raster * p.num_tb;
  const int g = u / per_group;
  const int first = g * p.raster;
  const int rows = min(p.num_cb - first, p.raster);
  const int r = u - g * per_group;
  cb = first + r % rows;
  tb = r / rows;
}

template <int CG, int BN, typename T>
__global__ void __launch_bounds__(kThreads, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w,   // weights: channels x K
                 const __grid_constant__ CUtensorMap tmap_t,   // tokens x K
                 const __grid_constant__ CUtensorMap tmap_d,   // D, for the staged epilogue
                 const __grid_constant__ Int8Params p) {
  constexpr int TROWS = BN / CG;                    // token rows each CTA of a pair loads
  constexpr int CW = BN < 32 ? BN : 32;             // tokens per epilogue chunk
  constexpr int NCH = BN / CW;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw_base);

  const uint32_t bars = base + p.bars_offset;
  const uint32_t full_bar = bars;                        // [stages]
  const uint32_t empty_bar = bars + 8u * kMaxStages;     // [stages]
  const uint32_t tfull_bar = bars + 16u * kMaxStages;    // [2]
  const uint32_t tempty_bar = tfull_bar + 16u;           // [2]
  const uint32_t drain_bar = tempty_bar + 16u;
  const uint32_t tmem_slot = drain_bar + 8u;
  const uint32_t abort_flag = tmem_slot + 4u;

  const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const uint32_t lane = threadIdx.x & 31u;
  const bool split = CG == 1 && p.split > 1;
  const uint32_t rank = (CG == 2 || split) ? cluster_ctarank() : 0u;
  const bool leader = CG == 1 || rank == 0;
  const int slot0 = CG == 2 ? (int)(blockIdx.x / 2) : (split ? (int)(blockIdx.x / p.split) : (int)blockIdx.x);
  const int slots = CG == 2 ? (int)(gridDim.x / 2) : (split ? p.num_units : (int)gridDim.x);
  const int kb_begin = split ? (int)rank * p.num_kb / p.split : 0;
  const int kb_end = split ? ((int)rank + 1) * p.num_kb / p.split : p.num_kb;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_t);
    if (p.stg_bufs > 0) prefetch_tmap(&tmap_d);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar + 8u * s, 1);
      mbar_init(empty_bar + 8u * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8u * a, 1);
      mbar_init(tempty_bar + 8u * a, 4 * CG);
    }
    mbar_init(drain_bar, 1);
    st_shared_u32(abort_flag, 0u);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<CG>(tmem_slot, (uint32_t)p.tmem_cols);
    tmem_relinquish<CG>();
  }
  tc_fence_before();
  if constexpr (CG == 2) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu,
      *reinterpret_cast<volatile uint32_t*>(base_ptr + (tmem_slot - base)), 0);

  SharedCtl ctl;
  ctl.abort_addr = abort_flag;
  ctl.abort_peer = CG == 2 ? mapa_shared(abort_flag, rank ^ 1u) : 0u;
  ctl.timeout_ns = p.timeout_ns;
  ctl.status = p.status;

  // Until here nothing of this launch depended on the kernels before it.  In the
  // linear layer only the tokens do (the weights were complete before the
  // quantisation of the tokens began): the producer then fetches the first
  // weights before it waits.
  if (!(warp == 0 && p.weights_ready)) {
    grid_dependency_wait();
    grid_launch_dependents();
  }

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (p.flags & GEMM_FLAG_INJECT_STALL) {
      if (p.weights_ready) grid_dependency_wait();
    } else {
      const uint32_t issue = elect_one() ? 1u : 0u;
      const uint64_t policy = policy_evict_normal();
      const uint32_t leader_full = CG == 2 ? mapa_shared(full_bar, 0) : full_bar;
      const uint32_t tx_bytes = p.stage_bytes * CG;
      int stage = 0;
      uint32_t phase = 0, issued_mask = 0, issued_parity = 0;
      bool ok = true;
      int ahead = 0;      // k-blocks of the first tile whose weights are on their way
      if (p.weights_ready) {
        int cb, tb;
        tile_coords(slot0, p, cb, tb);
        const int32_t c0 = (cb * CG + (int32_t)(CG == 2 ? rank : 0u)) * kChannels;
        ahead = min(p.stages, kb_end - kb_begin);
        for (int s = 0; s < ahead; ++s) {
          if (CG == 1 || issue) {
            mbar_arrive_expect_tx(full_bar + 8u * s, tx_bytes, leader ? issue : 0u);
            const uint32_t w_dst = base + (uint32_t)s * p.stage_bytes, target = leader_full + 8u * s;
            if constexpr (CG == 2) tma_load_2d_pair(w_dst, &tmap_w, target, (kb_begin + s) * kAtom, c0, policy, issue);
            else tma_load_2d(w_dst, &tmap_w, target, (kb_begin + s) * kAtom, c0, policy, issue);
          }
        }
        __syncwarp();
        grid_dependency_wait();
        grid_launch_dependents();
      }
      for (int u = slot0; u < p.num_units && ok; u += slots) {
        int cb, tb;
        tile_coords(u, p, cb, tb);
        const int32_t c0 = (cb * CG + (int32_t)(CG == 2 ? rank : 0u)) * kChannels;
        const int32_t t0 = tb * BN + (CG == 2 ? (int32_t)rank * TROWS : 0);
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_test_wait(empty_bar + 8u * stage, phase ^ 1u)) {
            const bool w = wait_bar<false>(empty_bar + 8u * stage, phase ^ 1u, ctl, ROLE_PRODUCER, stage);
            if (!__all_sync(__activemask(), w)) { ok = false; break; }
          }
          const uint32_t w_dst = base + (uint32_t)stage * p.stage_bytes;
          const uint32_t t_dst = w_dst + p.a_bytes;
          const uint32_t target = leader_full + 8u * stage;
          if (CG == 1 || issue) {
            const uint32_t weights = ahead == 0 ? issue : 0u;
            mbar_arrive_expect_tx(full_bar + 8u * stage, tx_bytes, leader ? weights : 0u);
            if constexpr (CG == 2) {
              tma_load_2d_pair(w_dst, &tmap_w, target, kb * kAtom, c0, policy, weights);
              tma_load_2d_pair(t_dst, &tmap_t, target, kb * kAtom, t0, policy, issue);
            } else {
              tma_load_2d(w_dst, &tmap_w, target, kb * kAtom, c0, policy, weights);
              tma_load_2d(t_dst, &tmap_t, target, kb * kAtom, t0, policy, issue);
            }
          }
          if (ahead > 0) --ahead;
          issued_mask |= 1u << stage;
          issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (!ok && leader) {
        // Let every load already issued land before the CTA may exit (a pair
        // leader's barriers cover its peer's loads too).
        for (int s = 0; s < p.stages; ++s)
          if (issued_mask & (1u << s)) drain_wait(full_bar + 8u * s, (issued_parity >> s) & 1u, 100000000ull);
      } else if (!ok) {
        const uint64_t t0 = globaltimer_ns();   // pair peer: a short fixed window before the teardown barrier
        while (globaltimer_ns() - t0 < 2000000ull) {}
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (leader) {
      const uint32_t issue = elect_one() ? 1u : 0u;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true, issued = false;
      for (int u = slot0; u < p.num_units && ok; u += slots) {
        const bool wt = wait_bar<CG == 2>(tempty_bar + 8u * acc, acc_phase ^ 1u, ctl, ROLE_MMA, 0x80u | acc);
        if (!__all_sync(0xffffffffu, wt)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        bool ready = false;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          const bool w = ready || wait_bar<CG == 2>(full_bar + 8u * stage, phase, ctl, ROLE_MMA, stage);
          if (!w) { ok = false; break; }
          tc_fence_after();
          const uint32_t w_src = base + (uint32_t)stage * p.stage_bytes;
          if (CG == 1 || issue) {
            const uint64_t wd = sw128_kmajor_desc(w_src), td = sw128_kmajor_desc(w_src + p.a_bytes);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_i8<CG>(d_tmem, wd + 2u * kk, td + 2u * kk, p.idesc, (kb != kb_begin || kk) ? 1u : 0u, issue);
            if constexpr (CG == 2) mma_commit_pair(empty_bar + 8u * stage, 0x3, issue);
            else mma_commit(empty_bar + 8u * stage, issue);
          }
          issued = true;
          if (++stage == p.stages) { stage = 0; phase ^= 1u; }
          ready = CG == 2 ? mbar_test_wait_cluster(full_bar + 8u * stage, phase)
                          : mbar_test_wait(full_bar + 8u * stage, phase);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if constexpr (CG == 2) mma_commit_pair(tfull_bar + 8u * acc, 0x3, issue);
        else mma_commit(tfull_bar + 8u * acc, issue);
        if (++acc == p.num_acc) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok && issued) {
        if constexpr (CG == 2) mma_commit_pair(drain_bar, 0x1, issue);
        else mma_commit(drain_bar, issue);
        drain_wait(drain_bar, 0, 100000000ull);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const uint32_t q = warp & 3u;                        // TMEM lane quadrant
    const int row = (int)(32u * q + lane);               // channel within the CTA's 128
    const uint32_t gtid = (warp - 2u) * 32u + lane;
    const bool issuer = gtid == 0;
    const uint32_t stg = base + p.stg_offset;
    const uint32_t sa_s = base + p.sa_offset + q * (uint32_t)(BN * 4);   // this warp's copy of the token scales
    const uint32_t leader_tempty = CG == 2 ? mapa_shared(tempty_bar, 0) : tempty_bar;
    const uint64_t key = p.drop.on ? drop_key(p.drop) : 0;
    uint32_t chunk_no = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int u = slot0; u < p.num_units; u += slots) {
      int cb, tb;
      tile_coords(u, p, cb, tb);
      const int c0 = (cb * CG + (int)(CG == 2 ? rank : 0u)) * kChannels;
      const int t0 = tb * BN;
      const int ch = c0 + row;
      const bool ch_ok = ch < p.n;
      const float sb = ch_ok ? (p.sb ? p.sb[ch] : 1.f) : 0.f;
      const float bias = ch_ok && p.bias ? load_as_f32(p.bias, p.bias_type, ch) : 0.f;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < (BN + 31) / 32; ++i) {
        const int t = i * 32 + (int)lane;
        if (t < BN) st_shared_u32(sa_s + 4u * t, __float_as_uint(t0 + t < p.m ? (p.sa ? p.sa[t0 + t] : 1.f) : 0.f));
      }
      __syncwarp();
      const bool ok = wait_bar<false>(tfull_bar + 8u * acc, acc_phase, ctl, ROLE_EPILOGUE, acc);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((32u * q) << 16) + (uint32_t)(acc * BN);
      if (split) {
        // This CTA's partial tile, [token][channel] int32, over the ring: every
        // load has landed and every MMA has read it.
#pragma unroll 1
        for (int i = 0; i < NCH; ++i) {
          uint32_t r[CW];
          if constexpr (CW == 32) tmem_ld32(t_row + (uint32_t)(i * CW), r); else tmem_ld16(t_row + (uint32_t)(i * CW), r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < CW; ++j) st_shared_u32(base + (uint32_t)(((i * CW + j) * kChannels + row) * 4), r[j]);
        }
        break;   // one tile per cluster; the sum follows the cluster barrier
      }
#pragma unroll 1
      for (int i = 0; i < NCH; ++i) {
        uint32_t r[CW];
        if constexpr (CW == 32) tmem_ld32(t_row + (uint32_t)(i * CW), r); else tmem_ld16(t_row + (uint32_t)(i * CW), r);
        tmem_ld_wait();
        if (i == NCH - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(leader_tempty + 8u * acc); else mbar_arrive(tempty_bar + 8u * acc);
          }
        }
        const int tc = t0 + i * CW;
        float v[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) v[j] = finish((int32_t)r[j], ld_shared_f32(sa_s + 4u * (uint32_t)(i * CW + j)), sb, bias);
        if (p.drop.on) {
          const int64_t index = drop_index(p.drop, tc, ch);
#pragma unroll
          for (int j = 0; j < CW; ++j)
            v[j] = drop_keeps(key, p.drop.threshold, index + j * p.drop.row_elems) ? v[j] * p.drop.grow : 0.f;
        }
        if (p.c && ch_ok) {
          const T* c = static_cast<const T*>(p.c) + (int64_t)tc * p.ldc + ch;
          float cv[CW];
#pragma unroll
          for (int j = 0; j < CW; ++j) cv[j] = tc + j < p.m ? to_f32(c[j * p.ldc]) : 0.f;
#pragma unroll
          for (int j = 0; j < CW; ++j) v[j] += cv[j];
        }
        if (p.stg_bufs > 0) {
          const uint32_t buf = stg + (p.stg_bufs == 2 ? (chunk_no & 1u) : 0u) * p.stg_bytes;
          if (issuer) {
            if (p.stg_bufs == 2) bulk_wait_group_read<1>(); else bulk_wait_group_read<0>();
          }
          named_bar_sync(1, 128);
#pragma unroll
          for (int j = 0; j < CW; ++j) {
            const T o = from_f32<T>(v[j]);
            const uint32_t at = buf + (uint32_t)((j * kChannels + row) * (int)sizeof(T));
            if constexpr (sizeof(T) == 4) {
              st_shared_u32(at, __float_as_uint(v[j]));
            } else {
              uint16_t h;
              __builtin_memcpy(&h, &o, 2);
              st_shared_u16(at, h);
            }
          }
          fence_proxy_async_shared();
          named_bar_sync(1, 128);
          if (issuer) {
            if (tc < p.m && c0 < p.n) tma_store_2d(&tmap_d, buf, c0, tc);
            bulk_commit_group();
          }
          ++chunk_no;
        } else if (ch_ok) {
          T* d = static_cast<T*>(p.d) + (int64_t)tc * p.ldd + ch;
#pragma unroll
          for (int j = 0; j < CW; ++j)
            if (tc + j < p.m) d[j * p.ldd] = from_f32<T>(v[j]);
        }
      }
      if (++acc == p.num_acc) { acc = 0; acc_phase ^= 1u; }
    }
    if (issuer && p.stg_bufs > 0) bulk_wait_group<0>();
  }

  // ------------------------------------------------------------ split-K sum and teardown
  __syncwarp();
  tc_fence_before();
  if (split) {
    cluster_arrive();
    cluster_wait();
    if (warp >= 2) {
      // CTA `rank` finishes its share of the tokens: a warp takes a token, a lane
      // four channels, with every peer's 16 bytes in flight at once.
      int cb, tb;
      tile_coords(slot0, p, cb, tb);
      const int ch0 = cb * kChannels + 4 * (int)lane, t0 = tb * BN;
      const int per = BN / p.split;
      float sb[4], bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = ch0 + e < p.n;
        sb[e] = in && p.sb ? p.sb[ch0 + e] : 1.f;
        bias[e] = in && p.bias ? load_as_f32(p.bias, p.bias_type, ch0 + e) : 0.f;
      }
      const uint64_t key = p.drop.on ? drop_key(p.drop) : 0;
      for (int j = (int)rank * per + (int)warp - 2; j < (int)(rank + 1) * per; j += 4) {
        const int t = t0 + j;
        if (t >= p.m) break;
        const uint32_t at = base + (uint32_t)((j * kChannels + 4 * (int)lane) * 4);
        uint4 part[kMaxSplit];
#pragma unroll
        for (int s = 0; s < kMaxSplit; ++s) part[s] = s < p.split ? ld_shared_cluster_v4(mapa_shared(at, (uint32_t)s)) : make_uint4(0, 0, 0, 0);
        uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kMaxSplit; ++s) { sum[0] += part[s].x; sum[1] += part[s].y; sum[2] += part[s].z; sum[3] += part[s].w; }
        const float sa = p.sa ? p.sa[t] : 1.f;
        T* const d = static_cast<T*>(p.d) + (int64_t)t * p.ldd + ch0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (ch0 + e >= p.n) break;
          float v = finish((int32_t)sum[e], sa, sb[e], bias[e]);
          if (p.drop.on) v = drop_keeps(key, p.drop.threshold, drop_index(p.drop, t, ch0 + e)) ? v * p.drop.grow : 0.f;
          if (p.c) v += to_f32(static_cast<const T*>(p.c)[(int64_t)t * p.ldc + ch0 + e]);
          d[e] = from_f32<T>(v);
        }
      }
      __syncwarp();
    }
    cluster_arrive();
    cluster_wait();   // peers may still read this CTA's partial tile
  } else if constexpr (CG == 2) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, (uint32_t)p.tmem_cols);
  }
}

// ----------------------------------------------------------------- host
struct Resolved {
  int cg, bn, split, stages, max_stages;
  int grid, num_sms;
  int64_t smem_bytes;
  Int8Params p;
  char reason[128];
};

#define FAIL(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_CANNOT_IMPLEMENT; } while (0)
#define BAD(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_BAD_ARGS; } while (0)

// `tokens`: A and its scales are read or written (not by the few-token form of the linear layer).
int check(const Int8GemmArgs* a, bool tokens, Resolved& r) {
  if (!a) BAD("null args");
  if (a->struct_size != sizeof(Int8GemmArgs)) BAD("Int8GemmArgs.struct_size %u != %zu", a->struct_size, sizeof(Int8GemmArgs));
  if (!type_ok(a->d_type)) FAIL("unknown d_type %d", a->d_type);
  if (a->bias && !type_ok(a->bias_type)) FAIL("unknown bias_type %d", a->bias_type);
  if (a->m < 0 || a->n < 0 || a->k <= 0) FAIL("empty problem %lld x %lld x %lld", (long long)a->m, (long long)a->n, (long long)a->k);
  if (a->m > INT32_MAX / 2 || a->n > INT32_MAX / 2) FAIL("dimension too large");
  if (a->k > 131071) FAIL("k %lld: the int32 sum is exact up to k = 131071", (long long)a->k);
  if (a->flags & ~(uint32_t)GEMM_FLAG_INJECT_STALL) FAIL("unknown flags 0x%x", a->flags);
  const char* why = "";
  if (drop_resolve(a->drop, a->m, a->n, r.p.drop, &why) != GEMM_OK) FAIL("%s", why);
  if (a->m > 0 && a->n > 0) {
    if ((tokens && !a->a) || !a->b || !a->d) BAD("null A/B/D pointer");
    const uintptr_t pa = tokens ? reinterpret_cast<uintptr_t>(a->a) : 0;
    const int64_t lda = tokens ? a->lda : a->ldb;
    if ((pa | reinterpret_cast<uintptr_t>(a->b)) & 15) FAIL("A/B must be 16-byte aligned");
    if (lda < a->k || a->ldb < a->k) FAIL("lda/ldb must be >= k");
    if ((lda | a->ldb) & 15) FAIL("lda/ldb must be multiples of 16");
    const uintptr_t e = (uintptr_t)type_bytes(a->d_type);
    if ((reinterpret_cast<uintptr_t>(a->d) | reinterpret_cast<uintptr_t>(a->c)) % e) FAIL("D/C must be aligned to their element");
    if (a->ldd < a->n) FAIL("ldd must be >= n");
    if (a->c && a->ldc < a->n) FAIL("ldc must be >= n");
    if ((reinterpret_cast<uintptr_t>(a->scale_a) | reinterpret_cast<uintptr_t>(a->scale_b)) & 3) FAIL("scales must be 4-byte aligned");
    if (a->bias && reinterpret_cast<uintptr_t>(a->bias) % type_bytes(a->bias_type)) FAIL("bias must be aligned to its element");
  }
  return GEMM_OK;
}

bool supported(int cg, int bn) {
  return cg == 1 ? (bn == 16 || bn == 32 || bn == 64 || bn == 128) : (bn == 128 || bn == 256);
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    sms = 148;
  }
  return sms;
}

// Tile and split from the sizes.
void choose(const Int8GemmArgs* a, int num_sms, int& cg, int& bn, int& split) {
  const int64_t cb = (a->n + 127) / 128;
  if (!bn && !cg && a->m > 128 && ((a->n + 255) / 256) * ((a->m + 255) / 256) * 2 >= num_sms) {
    cg = 2; bn = 256;
  }
  if (!cg) cg = 1;
  if (!bn) bn = cg == 2 ? 256 : a->m <= 16 ? 16 : a->m <= 32 ? 32 : a->m <= 64 ? 64 : 128;
  if (!split) {
    split = 1;
    if (cg == 1) {
      const int64_t tiles = cb * ((a->m + bn - 1) / bn);
      const int64_t kb = (a->k + kAtom - 1) / kAtom;
      while (split < 8 && tiles * split * 2 <= 2 * num_sms && kb >= split * 2 * 4) split *= 2;
    }
  }
}

int resolve(const Int8GemmArgs* a, Resolved& r) {
  memset(&r, 0, sizeof(r));
  const int rc = check(a, true, r);
  if (rc != GEMM_OK) return rc;
  r.num_sms = sm_count();
  r.cg = a->cta_group; r.bn = a->tile_n; r.split = a->split_k;
  choose(a, r.num_sms, r.cg, r.bn, r.split);
  if (r.cg != 1 && r.cg != 2) FAIL("cta_group must be 1 or 2");
  if (!supported(r.cg, r.bn)) FAIL("tile_n %d unsupported for cta_group %d", r.bn, r.cg);
  if (r.split != 1 && r.split != 2 && r.split != 4 && r.split != 8) FAIL("split_k must be 1, 2, 4 or 8");
  Int8Params& p = r.p;
  p.num_kb = (int)((a->k + kAtom - 1) / kAtom);
  if (r.split > 1) {
    if (r.cg != 1) FAIL("split_k needs cta_group 1");
    if (r.split > p.num_kb) FAIL("split_k %d of %d K blocks", r.split, p.num_kb);
  }
  p.split = r.split;
  p.d = a->d; p.ldd = a->ldd; p.c = a->c; p.ldc = a->ldc;
  p.sa = a->scale_a; p.sb = a->scale_b; p.bias = a->bias; p.bias_type = a->bias_type;
  p.m = (int32_t)a->m; p.n = (int32_t)a->n;
  p.num_cb = (int)((a->n + kChannels * r.cg - 1) / (kChannels * r.cg));
  p.num_tb = (int)((a->m + r.bn - 1) / r.bn);
  if ((int64_t)p.num_cb * p.num_tb > INT32_MAX / 16) FAIL("too many tiles");
  p.num_units = p.num_cb * p.num_tb;
  p.raster = p.num_cb < 4 ? (p.num_cb > 0 ? p.num_cb : 1) : 4;
  p.a_bytes = kChannels * kAtom;
  p.stage_bytes = p.a_bytes + (uint32_t)(r.bn / r.cg) * kAtom;
  p.num_acc = r.split > 1 ? 1 : 2;
  int cols = 32;
  while (cols < p.num_acc * r.bn) cols *= 2;
  p.tmem_cols = cols;
  p.idesc = make_idesc(kChannels * r.cg, r.bn);
  // Shared memory: ring, barriers, staging (whole-K form, when D allows TMA stores), token scales.
  const int e = type_bytes(a->d_type);
  const int cw = r.bn < 32 ? r.bn : 32;
  p.stg_bytes = (uint32_t)(cw * kChannels * e);
  // (A TMA store whose row extent ends inside 16 bytes writes the rest of them too.)
  p.stg_bufs = r.split == 1 && a->m > 0 && rows_16b(a->d, a->ldd, e) && (a->n * e) % 16 == 0 ? 2 : 0;
  const int64_t fixed = 1024 + kBarrierBytes + (int64_t)p.stg_bufs * p.stg_bytes + 4 * r.bn * 4;
  r.max_stages = (int)((kSmemLimit - fixed) / p.stage_bytes);
  if (r.max_stages > 12) r.max_stages = 12;
  const int kb_cta = (p.num_kb + r.split - 1) / r.split;
  r.stages = r.max_stages;
  if (r.split > 1) {
    if (r.stages > kb_cta) r.stages = kb_cta;
    while ((int64_t)r.stages * p.stage_bytes < (int64_t)r.bn * kChannels * 4) ++r.stages;   // the partial tile lies over the ring
  }
  p.stages = r.stages;
  p.bars_offset = (uint32_t)r.stages * p.stage_bytes;
  p.stg_offset = p.bars_offset + kBarrierBytes;
  p.sa_offset = p.stg_offset + (uint32_t)p.stg_bufs * p.stg_bytes;
  r.smem_bytes = 1024 + (int64_t)p.sa_offset + 4 * r.bn * 4;
  p.status = a->status;
  p.timeout_ns = (uint64_t)(a->timeout_ms ? a->timeout_ms : 4000u) * 1000000ull;
  p.flags = a->flags;
  const int64_t slots = r.split > 1 ? p.num_units : (r.num_sms / r.cg < p.num_units ? r.num_sms / r.cg : p.num_units);
  r.grid = (int)(slots * (r.split > 1 ? r.split : r.cg));
  return GEMM_OK;
}
#undef FAIL
#undef BAD

using KernelFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, Int8Params);

template <typename T>
KernelFn pick(int cg, int bn) {
  if (cg == 1) {
    switch (bn) {
      case 16: return int8_gemm_kernel<1, 16, T>;
      case 32: return int8_gemm_kernel<1, 32, T>;
      case 64: return int8_gemm_kernel<1, 64, T>;
      default: return int8_gemm_kernel<1, 128, T>;
    }
  }
  return bn == 128 ? int8_gemm_kernel<2, 128, T> : int8_gemm_kernel<2, 256, T>;
}

std::mutex g_attr_mu;
struct AttrSet { KernelFn fn; int dev; };
AttrSet g_attr_set[512];
int g_attr_n = 0;

bool ensure_smem_attr(KernelFn fn, int dev) {
  std::lock_guard<std::mutex> lock(g_attr_mu);
  for (int i = 0; i < g_attr_n; ++i)
    if (g_attr_set[i].fn == fn && g_attr_set[i].dev == dev) return true;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (g_attr_n < 512) g_attr_set[g_attr_n++] = {fn, dev};
  return true;
}

// Few tokens and no tile asked for: one launch without tensor cores.
bool use_gemv(const Int8GemmArgs& a, int num_sms) {
  return !a.tile_n && !a.cta_group && !a.split_k && !a.flags && gemv_fits(a.m, a.n, a.k, num_sms);
}

int launch_gemv(const Int8GemmArgs& a, const void* x, int32_t x_type, int64_t ldx, int num_sms, cudaStream_t st) {
  GemvParams g;
  memset(&g, 0, sizeof(g));
  const char* why = "";
  if (drop_resolve(a.drop, a.m, a.n, g.drop, &why) != GEMM_OK) return GEMM_ERR_CANNOT_IMPLEMENT;
  g.x = x; g.ldx = ldx; g.x_type = x_type;
  g.b = static_cast<const int8_t*>(a.b); g.ldb = a.ldb;
  g.d = a.d; g.ldd = a.ldd; g.d_type = a.d_type; g.c = a.c; g.ldc = a.ldc;
  g.sa = a.scale_a; g.sb = a.scale_b; g.bias = a.bias; g.bias_type = a.bias_type;
  g.m = (int32_t)a.m; g.n = (int32_t)a.n; g.k = (int32_t)a.k;
  g.status = a.status;
  g.timeout_ns = (uint64_t)(a.timeout_ms ? a.timeout_ms : 4000u) * 1000000ull;
  g.wide = x_type != kTypeInt8 && rows_16b(x, ldx, type_bytes(x_type));
  if (gemv_launch(g, num_sms, st) != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}

// One product; the device of D is current.  `weights_ready`: the kernel launched
// just before on this stream writes neither the weights nor anything they depend on.
int launch_product(const Int8GemmArgs& a, bool weights_ready, cudaStream_t st, int dev) {
  Resolved r;
  const int rc = resolve(&a, r);
  if (rc != GEMM_OK) return rc;
  if (!get_encode()) return GEMM_ERR_LAUNCH;
  CUtensorMap tw, tt, td;
  if (!encode_2d(&tw, a.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)a.k, (uint64_t)a.n, (uint64_t)a.ldb, kAtom, kChannels, 128) ||
      !encode_2d(&tt, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)a.k, (uint64_t)a.m, (uint64_t)a.lda, kAtom,
                 (uint32_t)(r.bn / r.cg), 128))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  memset(&td, 0, sizeof(td));
  if (r.p.stg_bufs > 0) {
    const CUtensorMapDataType t = a.d_type == GEMM_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : a.d_type == GEMM_TYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if (!encode_2d(&td, a.d, t, (uint64_t)a.n, (uint64_t)a.m, (uint64_t)(a.ldd * type_bytes(a.d_type)), kChannels,
                   (uint32_t)(r.bn < 32 ? r.bn : 32), 0))
      return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  KernelFn fn = a.d_type == GEMM_TYPE_BF16 ? pick<__nv_bfloat16>(r.cg, r.bn)
              : a.d_type == GEMM_TYPE_FP16 ? pick<__half>(r.cg, r.bn) : pick<float>(r.cg, r.bn);
  if (!ensure_smem_attr(fn, dev)) return GEMM_ERR_LAUNCH;
  r.p.weights_ready = weights_ready ? 1 : 0;
  if (launch_overlapped(fn, dim3((unsigned)r.grid), dim3(kThreads), (size_t)r.smem_bytes, r.split > 1 ? r.split : r.cg, st,
                        tw, tt, td, r.p) != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}

}  // namespace

extern "C" int gemm_sm100a_int8_query(const Int8GemmArgs* args, GemmInfo* info) {
  Resolved r;
  const int rc = resolve(args, r);
  if (info) {
    memset(info, 0, sizeof(*info));
    info->struct_size = sizeof(GemmInfo);
    info->tile_m = kChannels * r.cg; info->tile_n = r.bn; info->tile_k = kAtom; info->stages = r.stages;
    info->cta_group = r.cg; info->cluster_m = r.split > 1 ? r.split : r.cg; info->max_stages = r.max_stages;
    info->smem_bytes_per_stage = r.p.stage_bytes; info->smem_bytes = r.smem_bytes;
    info->tmem_columns = r.p.tmem_cols; info->grid_ctas = r.grid; info->num_tiles = r.p.num_units;
    info->num_sms = r.num_sms; info->can_implement = rc == GEMM_OK;
    memcpy(info->reason, r.reason, sizeof(info->reason));
    info->epilogue_staging_buffers = r.p.stg_bufs;
  }
  return rc;
}

extern "C" int gemm_sm100a_int8_launch(const Int8GemmArgs* args, void* stream) {
  Resolved r;
  memset(&r, 0, sizeof(r));
  const int rc = check(args, true, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(args->d);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const int sms = sm_count();
  if (use_gemv(*args, sms)) return launch_gemv(*args, args->a, kTypeInt8, args->lda, sms, st);
  return launch_product(*args, false, st, guard.dev);
}

extern "C" int gemm_sm100a_int8_linear(const Int8GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream) {
  Resolved r;
  memset(&r, 0, sizeof(r));
  const int sms = sm_count();
  const bool few = args && args->struct_size == sizeof(Int8GemmArgs) && use_gemv(*args, sms);
  const int rc = check(args, !few, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  if (!type_ok(x_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!x || (!few && !args->scale_a)) return GEMM_ERR_BAD_ARGS;
  if (ldx < args->k || reinterpret_cast<uintptr_t>(x) % type_bytes(x_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(args->d);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  if (few) return launch_gemv(*args, x, x_type, ldx, sms, st);
  Int8QuantArgs q;
  memset(&q, 0, sizeof(q));
  q.struct_size = sizeof(q);
  q.x_type = x_type; q.rows = args->m; q.cols = args->k; q.x = x; q.ldx = ldx;
  q.q = const_cast<void*>(args->a); q.ldq = args->lda; q.scale = const_cast<float*>(args->scale_a);
  const int rq = gemm_sm100a_quantize_int8(&q, stream);
  return rq != GEMM_OK ? rq : launch_product(*args, true, st, guard.dev);
}
