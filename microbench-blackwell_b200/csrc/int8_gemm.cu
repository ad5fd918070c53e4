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
// warps 2..5 run the epilogue (one TMEM lane quadrant each; in a pair with a short
// main loop warps 6..9 take every other chunk).
//
// Measured on B200 (1000 W cap): 8192 x 8192 x 8192 in 344 us under ncu, tensor pipe
// 96 % active, 3.19 PFLOP/s, and in 361 us back to back; 8192 x 28672 x 8192 back to back
// 1.39 ms, 2.77 PFLOP/s at the clock that the power cap leaves.  One token x 8192 x 8192 in
// 14.5 us (from a graph), 4.6 of the 6.55 TB/s that a copy reaches; about 4 us of it are
// launch, first loads and last stores (a 1024 x 1024 layer takes 4.8 us in all).
//   whole-K form   persistent CTAs (CTA pairs for large problems), two
//                  accumulators, so a tile's epilogue overlaps the next mainloop.
//   split-K form   for few tiles: the CTAs of a cluster share one tile's K and
//                  add their int32 partial tiles through distributed shared
//                  memory (exact, so the order does not matter); no workspace.
//   fused form     for a linear layer of at most 8 tokens, in one launch: while the
//                  ring fills with weights, 12 warps find the tokens' maxima and
//                  quantise the CTA's part of them straight into the swizzled
//                  operand, which stays in shared memory for all of its tiles.
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
#include "tensor_map.cuh"

using namespace sm100;
using namespace int8op;

namespace {

constexpr int kFusedTokens = 8;         // most tokens of the fused form: one 8-row group of the swizzle
constexpr int kFusedBN = 16;            // its MMA N, the smallest there is for 128 channels
constexpr int kStageWarps = 12;         // warps of the fused form that quantise tokens (the epilogue's four among them)
constexpr int kFusedElems = 16384;      // most tokens x K of the fused form (at most 128 KB of shared memory)
constexpr int kMaxGroups = 2;           // epilogue groups of a CTA pair's kernel (four warps each)
// Most threads of a CTA.
__host__ __device__ constexpr int threads_for(int cg, bool fuse) {
  return 64 + (fuse ? 32 * kStageWarps : 128 * (cg == 2 ? kMaxGroups : 1));
}
constexpr int kSmemLimit = 232448;      // 227 KiB of opt-in dynamic shared memory per CTA
// More than half of an SM's 228 KiB: at most one CTA of these kernels, or of the floating product's,
// per SM.  A CTA waits for tensor memory without a limit, and those of a pair or a split for one another:
// two kernels of different streams that share two SMs could each hold what the other one's CTA waits for.
constexpr int kMinSmemPerCta = 120 * 1024;
constexpr int kBarrierBytes = 1024;
constexpr int kStaticSmem = 512;        // bound of the static shared memory of the fused form
constexpr int kMaxStages = 32;
constexpr int kCBufs = 4;               // most staging buffers of an epilogue group that reads C by TMA:
                                        // all but two hold chunks of C on their way
constexpr int kAtom = 128;              // bytes (= K elements) of one swizzled K atom
constexpr uint32_t kTokAtom = 8 * kAtom;  // fused form: bytes of one K atom of the tokens
constexpr int kChannels = 128;          // channels per CTA
constexpr int kMaxSplit = 8;            // CTAs that may share a tile's K (portable cluster size)

template <int V>
struct IntC { static constexpr int value = V; };

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
  int32_t stg_bufs;                     // staging buffers (0: D is written from registers)
  int32_t tma_store;                    // D is written from them, by TMA
  int32_t groups;                       // epilogue groups: each takes every groups-th chunk of a tile
  int32_t c_bufs;                       // staging buffers of a group where C is staged
  int32_t c_staged;                     // chunks of C are fetched into the staging buffers (c_bufs per group)
  int32_t tmem_cols, num_acc;
  int32_t raster;                       // channel blocks per raster group
  uint32_t idesc;
  int32_t* status;
  uint64_t timeout_ns;
  uint32_t flags;
  const void* x; int64_t ldx;           // fused form: tokens before quantisation
  int32_t x_wide, k;
  uint32_t tok_offset;                  // fused form: quantised tokens, kTokAtom bytes per K atom
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

// Fused form: all staging warps, `tid` in [0, 32 * kStageWarps).  x's rows are
// read twice (the second time from L1); atoms [kb_begin, kb_end) of the quantised
// rows go to `tok`, 128-byte rows in the 128-byte swizzle, their scales to `sa_s`.
// Rows from m on and bytes beyond K stay undefined: those accumulator columns
// are not read, and the weights beyond K are zeros.  (Rows 8 to 15 of the MMA's
// operand are the next K atom's, after the last one the 1 KB behind it.)
template <typename X>
__device__ __forceinline__ void stage_tokens(const Int8Params& p, uint32_t tok, uint32_t sa_s, RowScale* rows, uint32_t* top,
                                             int kb_begin, int kb_end, int tid) {
  constexpr int V = Vec<X>::N, N = 32 * kStageWarps;
  constexpr int UN = 4;               // vectors in flight per thread, of whichever tokens they are
  const X* const x = static_cast<const X*>(p.x);
  const int nvec = (p.k + V - 1) / V;
  // Thread `tid` takes vectors tid, tid + N, ... of the m x `width` vectors from `first`.
  auto walk = [&](int first, int width, auto&& body) {
    const int total = p.m * width;
    const int dt = N / width, de = N - dt * width;
    int t = tid / width, e = tid - t * width;
    for (int i0 = tid & ~31; i0 < total; i0 += UN * N) {        // whole warps
      Vec<X> v[UN];
      int tt[UN], ee[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        tt[u] = t;
        ee[u] = first + e;
        v[u] = load_vec<X>(x + t * p.ldx + ee[u] * V, t < p.m ? p.k - ee[u] * V : 0, p.x_wide);
        t += dt;
        e += de;
        if (e >= width) { e -= width; ++t; }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i0 + u * N < total) body(tt[u], ee[u], v[u]);
    }
  };
  if (tid < kFusedTokens) top[tid] = 0u;
  __syncwarp();
  named_bar_sync(2, N);
  walk(0, nvec, [&](int t, int e, const Vec<X>& v) {
    // One shared atomic per warp where its vectors are of one token.
    uint32_t m = vec_magnitude<X>(v);
    t = min(t, p.m - 1);
    if (__all_sync(0xFFFFFFFFu, t == __shfl_sync(0xFFFFFFFFu, t, 0))) {
      m = __reduce_max_sync(0xFFFFFFFFu, m);
      if ((tid & 31) == 0) atomicMax(&top[t], m);
    } else {
      atomicMax(&top[t], m);
    }
  });
  __syncwarp();
  named_bar_sync(2, N);
  if (tid < p.m) {
    rows[tid] = row_scale(top[tid]);
    st_shared_u32(sa_s + 4u * tid, __float_as_uint(rows[tid].scale));
  }
  __syncwarp();
  named_bar_sync(2, N);
  const int e0 = kb_begin * (kAtom / V), e1 = min(nvec, kb_end * (kAtom / V));
  walk(e0, e1 - e0, [&](int t, int e, const Vec<X>& v) {
    if (t >= p.m) return;
    uint32_t w[V / 4];
    quantize_vec<X>(v, rows[t], w);
    const uint32_t b = (uint32_t)(e - e0) * V;                         // byte of the CTA's part of the row
    const uint32_t at = tok + (uint32_t)t * 128u + (b >> 7) * kTokAtom + ((((b >> 4) & 7u) ^ (uint32_t)t) << 4) + (b & 15u);
    if constexpr (V == 8) st_shared_v2(at, w[0], w[1]);
    else st_shared_u32(at, w[0]);
  });
}

// One element of a staged chunk.
template <typename T>
__device__ __forceinline__ float staged(uint32_t addr) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(ld_shared_u32(addr));
  } else {
    const uint16_t h = ld_shared_u16(addr);
    T v;
    __builtin_memcpy(&v, &h, 2);
    return to_f32(v);
  }
}

// A thread's column of a chunk, `tokens` rows of D from `d`, `step` bytes apart: for
// a D that TMA cannot store.  With one warp per scheduler every instruction counts, hence the running
// pointer and the paired conversions (777 x 5001 x 2048: 18.1 us through shared memory in
// aligned 16-byte stores).
template <typename T, int CW>
__device__ __forceinline__ void store_column(uint8_t* d, int64_t step, const float (&v)[CW], int tokens) {
#pragma unroll
  for (int j = 0; j < CW; j += 2) {
    uint8_t* const d1 = d + step;
    if constexpr (sizeof(T) == 4) {
      if (j < tokens) *reinterpret_cast<float*>(d) = v[j];
      if (j + 1 < tokens) *reinterpret_cast<float*>(d1) = v[j + 1];
    } else {
      const uint32_t h = pack2<T>(v[j], v[j + 1]);
      if (j < tokens) *reinterpret_cast<uint16_t*>(d) = (uint16_t)h;
      if (j + 1 < tokens) *reinterpret_cast<uint16_t*>(d1) = (uint16_t)(h >> 16);
    }
    d = d1 + step;
  }
}

template <int CG, int BN, typename T, bool FUSE>
__global__ void __launch_bounds__(threads_for(CG, FUSE), 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w,   // weights: channels x K
                 const __grid_constant__ CUtensorMap tmap_t,   // tokens x K
                 const __grid_constant__ CUtensorMap tmap_d,   // D, for the staged epilogue
                 const __grid_constant__ CUtensorMap tmap_c,   // C, where it is staged too
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
  const uint32_t tok_bar = abort_flag + 4u;              // fused form: the tokens are in place
  const uint32_t c_bar = tok_bar + 8u;                   // [groups][kCBufs]: a chunk of C is in its buffer
  const uint32_t lost_flag0 = c_bar + 8u * kCBufs * kMaxGroups;   // [groups]: a warp of the group has given up a wait
  __shared__ RowScale tok_rows[FUSE ? kFusedTokens : 1];
  __shared__ uint32_t tok_top[FUSE ? kFusedTokens : 1];

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
    if (p.tma_store) prefetch_tmap(&tmap_d);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar + 8u * s, 1);
      mbar_init(empty_bar + 8u * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8u * a, 1);
      mbar_init(tempty_bar + 8u * a, 4 * CG * p.groups);
    }
    mbar_init(drain_bar, 1);
    mbar_init(tok_bar, kStageWarps);
    for (int b = 0; b < kCBufs * kMaxGroups; ++b) mbar_init(c_bar + 8u * b, 1);
    st_shared_u32(abort_flag, 0u);
    for (int g = 0; g < kMaxGroups; ++g) st_shared_u32(lost_flag0 + 4u * g, 0u);
    fence_mbar_init();
  }
  __syncwarp();   // here and below: barriers and tensor memory instructions need a warp's lanes together
  if constexpr (CG == 2) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }
  // Until here nothing of this launch depended on the kernels before it, and it holds
  // no tensor memory while it waits for them (one of them might still need some).
  grid_dependency_wait();
  uint32_t tmem_base = 0;
  auto read_tmem_base = [&]() {
    tmem_base = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(base_ptr + (tmem_slot - base)), 0);
  };
  if (warp == 1) {
    tmem_alloc<CG>(tmem_slot, (uint32_t)p.tmem_cols);
    tmem_relinquish<CG>();
    grid_launch_dependents();   // the next kernel's blocks come after this one's have their tensor memory
  }
  if constexpr (CG == 2) {
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    read_tmem_base();
  } else if (warp == 1) {
    // The loads are on their way meanwhile; only the epilogue waits for the address.
    __syncwarp();
    read_tmem_base();
    tc_fence_before();
    named_bar_arrive(3, 160);
  } else if (warp >= 2 && warp < 6) {
    named_bar_sync(3, 160);
    tc_fence_after();
    read_tmem_base();
  }

  SharedCtl ctl;
  ctl.abort_addr = abort_flag;
  ctl.abort_peer = CG == 2 ? mapa_shared(abort_flag, rank ^ 1u) : 0u;
  ctl.timeout_ns = p.timeout_ns;
  ctl.status = p.status;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (!(p.flags & GEMM_FLAG_INJECT_STALL)) {
      const uint32_t issue = elect_one() ? 1u : 0u;
      const uint64_t policy = policy_evict_normal();
      const uint32_t leader_full = CG == 2 ? mapa_shared(full_bar, 0) : full_bar;
      const uint32_t tx_bytes = p.stage_bytes * CG;
      int stage = 0;
      uint32_t phase = 0, issued_mask = 0, issued_parity = 0;
      bool ok = true;
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
            mbar_arrive_expect_tx(full_bar + 8u * stage, tx_bytes, leader ? issue : 0u);
            if constexpr (CG == 2) {
              tma_load_2d_pair(w_dst, &tmap_w, target, kb * kAtom, c0, policy, issue);
              tma_load_2d_pair(t_dst, &tmap_t, target, kb * kAtom, t0, policy, issue);
            } else {
              tma_load_2d(w_dst, &tmap_w, target, kb * kAtom, c0, policy, issue);
              if constexpr (!FUSE) tma_load_2d(t_dst, &tmap_t, target, kb * kAtom, t0, policy, issue);
            }
          }
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
      if constexpr (FUSE) {
        const bool wt = wait_bar<false>(tok_bar, 0, ctl, ROLE_MMA, 0x90u);
        ok = __all_sync(0xffffffffu, wt);
      }
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
            const uint64_t wd = sw128_kmajor_desc(w_src);
            const uint64_t td = sw128_kmajor_desc(FUSE ? base + p.tok_offset + (uint32_t)(kb - kb_begin) * kTokAtom : w_src + p.a_bytes);
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
    if constexpr (FUSE) {
      stage_tokens<T>(p, base + p.tok_offset, base + p.sa_offset, tok_rows, tok_top, kb_begin, kb_end, (int)threadIdx.x - 64);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(tok_bar);
    }
    if (!FUSE || warp < 6) {
    // ------------------------------------------------------------ epilogue
    const uint32_t q = warp & 3u;                        // TMEM lane quadrant
    const int row = (int)(32u * q + lane);               // channel within the CTA's 128
    const uint32_t grp = CG == 2 ? (warp - 2u) >> 2 : 0u;
    const int groups = CG == 2 ? p.groups : 1;
    const bool issuer = ((warp - 2u) & 3u) * 32u + lane == 0;
    const uint32_t bar_id = grp ? 4u : 1u;               // named barrier of the group
    const uint32_t stg = base + p.stg_offset + grp * (uint32_t)p.stg_bufs * p.stg_bytes;
    const uint32_t lost_flag = lost_flag0 + 4u * grp;
    const uint32_t c_full = c_bar + grp * 8u * kCBufs;
    const uint32_t sa_s = base + p.sa_offset + (FUSE ? 0u : (warp - 2u) * (uint32_t)(BN * 4));   // this warp's copy of the token scales
    const uint32_t leader_tempty = CG == 2 ? mapa_shared(tempty_bar, 0) : tempty_bar;
    const uint64_t key = p.drop.on ? drop_key(p.drop) : 0;
    // Rows of an even length that begin at an even index: even channels are the first of a draw's pair.
    const bool drop_pairs = p.drop.on && !p.drop.all && !((p.drop.row_elems | p.drop.col0) & 1);
    const bool drop_odd_rows = p.drop.on && !p.drop.all && (p.drop.row_elems & 1);
    const uint64_t drop_step = (uint64_t)p.drop.row_elems * counter_rng::kGolden;   // two tokens on
    const uint32_t drop_thr = p.drop.threshold;
    const float drop_grow = p.drop.grow;
    uint32_t chunk_no = 0;
    // C staged: chunk x of this group (over all its tiles) goes through buffer x % c_bufs, is
    // replaced there by D, element by element in the same thread, and stored from it.  One
    // thread fetches c_bufs - 2 chunks ahead, also across tiles.
    const uint32_t c_bufs = (uint32_t)p.c_bufs;
    int c_u = slot0, c_i = (int)grp;
    uint32_t c_no = 0;
    const uint64_t c_policy = policy_evict_normal();
    auto fetch_c = [&]() {
      if (c_u >= p.num_units) return;
      int cb, tb;
      tile_coords(c_u, p, cb, tb);
      const uint32_t buf = c_no % c_bufs;
      mbar_arrive_expect_tx(c_full + 8u * buf, p.stg_bytes);
      tma_load_2d(stg + buf * p.stg_bytes, &tmap_c, c_full + 8u * buf,
                  (cb * CG + (int)(CG == 2 ? rank : 0u)) * kChannels, tb * BN + c_i * CW, c_policy);
      ++c_no;
      if ((c_i += groups) >= NCH) { c_i = (int)grp; c_u += slots; }
    };
    if (p.c_staged && issuer) {
      for (uint32_t b = 2; b < c_bufs; ++b) fetch_c();
    }
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
      bool large = false;    // one of the tile's tokens has a large scale
      if constexpr (!FUSE) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < (BN + 31) / 32; ++i) {
          const int t = i * 32 + (int)lane;
          const float sa = t < BN && t0 + t < p.m ? (p.sa ? p.sa[t0 + t] : 1.f) : 0.f;
          large |= is_large(sa);
          if (t < BN) st_shared_u32(sa_s + 4u * t, __float_as_uint(sa));
        }
        __syncwarp();
      } else {
        large = (int)lane < p.m && is_large(tok_rows[lane & (kFusedTokens - 1)].scale);
      }
      large = __any_sync(0xFFFFFFFFu, large);
      const bool ok = __all_sync(0xffffffffu, wait_bar<false>(tfull_bar + 8u * acc, acc_phase, ctl, ROLE_EPILOGUE, acc));
      if (!p.tma_store) {
        if (!ok) break;
      } else {
        // The warps meet at named barriers below, so after an abort all four leave, or none:
        // whichever gave up (here or on a chunk of C) says so before the first barrier, and
        // none can say so again before all have looked.
        if (!ok && lane == 0) st_shared_u32(lost_flag, 1u);
        __syncwarp();
        named_bar_sync(bar_id, 128);
        const bool lost = ld_shared_volatile_u32(lost_flag) != 0u;
        named_bar_sync(bar_id, 128);
        if (lost) break;
      }
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
      for (int i = (int)grp; i < NCH; i += groups) {
        __syncwarp();
        uint32_t r[CW];
        if constexpr (CW == 32) tmem_ld32(t_row + (uint32_t)(i * CW), r); else tmem_ld16(t_row + (uint32_t)(i * CW), r);
        tmem_ld_wait();
        if (i + groups >= NCH) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(leader_tempty + 8u * acc); else mbar_arrive(tempty_bar + 8u * acc);
          }
        }
        const int tc = t0 + i * CW;
        float v[CW];
        if (!large) {
#pragma unroll
          for (int j = 0; j < CW; j += 4) {
            const uint4 sa = ld_shared_v4(sa_s + 4u * (uint32_t)(i * CW + j));
            v[j] = finish((int32_t)r[j], __uint_as_float(sa.x), sb, bias);
            v[j + 1] = finish((int32_t)r[j + 1], __uint_as_float(sa.y), sb, bias);
            v[j + 2] = finish((int32_t)r[j + 2], __uint_as_float(sa.z), sb, bias);
            v[j + 3] = finish((int32_t)r[j + 3], __uint_as_float(sa.w), sb, bias);
          }
        } else {
#pragma unroll
          for (int j = 0; j < CW; ++j)
            v[j] = finish_large((int32_t)r[j], __uint_as_float(ld_shared_u32(sa_s + 4u * (uint32_t)(i * CW + j))), sb, bias);
        }
        if (p.drop.on) {
          const int64_t index = drop_index(p.drop, tc, ch);
          if (drop_pairs) {
            // Lanes 2 i and 2 i + 1 hold the two elements of a draw: the even lane draws for
            // token j, the odd one for token j + 1, and each passes on the other's word.
            const bool odd = lane & 1u;
            const uint64_t first = (uint64_t)(index + (odd ? p.drop.row_elems : 0)) >> 1;
            uint64_t z = key + (first + 1) * counter_rng::kGolden;
#pragma unroll
            for (int j = 0; j < CW; j += 2, z += drop_step) {
              const uint64_t h = counter_rng::mix64(z);
              const uint32_t lo = (uint32_t)h, hi = (uint32_t)(h >> 32);
              const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, odd ? lo : hi, 1);
              v[j] = (odd ? other : lo) >= drop_thr ? v[j] * drop_grow : 0.f;
              v[j + 1] = (odd ? hi : other) >= drop_thr ? v[j + 1] * drop_grow : 0.f;
            }
          } else if (drop_odd_rows) {
            // Rows of an odd length: of each two tokens, one (E) has its pairs at lanes 2 i, 2 i + 1 and
            // the other (O) at lanes 2 i + 1, 2 i + 2.  The lower lane of a pair draws for both, and
            // the upper one's word comes from one lane below; for lane 0, whose lower half would be in
            // the warp before, lane l draws the word of token pair l beforehand.
            const bool odd = lane & 1u;
            const int swap = (int)((p.drop.row0 + tc + p.drop.col0) & 1);      // 1: token j is O, j + 1 is E
            const uint64_t before = counter_rng::draw(key, (uint64_t)drop_index(p.drop, tc + 2 * ((int)lane % (CW / 2)) + 1 - swap,
                                                                                ch - (int)lane) >> 1) >> 32;
            const uint64_t first = (uint64_t)drop_index(p.drop, tc + (odd ? 1 - swap : swap), ch) >> 1;
            uint64_t z = key + (first + 1) * counter_rng::kGolden;
#pragma unroll
            for (int j = 0; j < CW; j += 2, z += drop_step) {
              const uint64_t h = counter_rng::mix64(z);
              const uint32_t own = (uint32_t)h;
              uint32_t below = __shfl_up_sync(0xFFFFFFFFu, (uint32_t)(h >> 32), 1);
              const uint32_t first_lane = __shfl_sync(0xFFFFFFFFu, (uint32_t)before, j / 2);
              if (lane == 0) below = first_lane;
              const bool e = odd == (swap != 0);                               // token j's word is the own one
              v[j] = (e ? own : below) >= drop_thr ? v[j] * drop_grow : 0.f;
              v[j + 1] = (e ? below : own) >= drop_thr ? v[j + 1] * drop_grow : 0.f;
            }
          } else {
#pragma unroll
            for (int j = 0; j < CW; ++j)
              v[j] = drop_keeps(p.drop, key, index + j * p.drop.row_elems) ? v[j] * drop_grow : 0.f;
          }
        }
        if (p.c && ch_ok && !p.c_staged) {
          const T* c = static_cast<const T*>(p.c) + (int64_t)tc * p.ldc + ch;
          float cv[CW];
#pragma unroll
          for (int j = 0; j < CW; ++j, c += p.ldc) cv[j] = tc + j < p.m ? to_f32(*c) : 0.f;
#pragma unroll
          for (int j = 0; j < CW; ++j) v[j] += cv[j];
        }
        if (p.tma_store) {
          const uint32_t b = p.c_staged ? chunk_no % c_bufs : chunk_no & 1u;
          const uint32_t buf = stg + b * p.stg_bytes;
          const uint32_t at = buf + (uint32_t)(row * (int)sizeof(T));
          if (p.c_staged) {
            if (issuer) {
              bulk_wait_group_read<1>();     // the buffer that fetch_c takes has been stored
              fetch_c();
            }
            __syncwarp();
            const bool c_ok = wait_bar<false>(c_full + 8u * b, (chunk_no / c_bufs) & 1u, ctl, ROLE_EPILOGUE, 0xC0u | b);
            if (!c_ok) st_shared_u32(lost_flag, 1u);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < CW; ++j) v[j] += staged<T>(at + (uint32_t)(j * kChannels * (int)sizeof(T)));
          } else {
            if (issuer) bulk_wait_group_read<1>();
            __syncwarp();
            named_bar_sync(bar_id, 128);
          }
#pragma unroll
          for (int j = 0; j < CW; j += 2) {
            if constexpr (sizeof(T) == 4) {
              st_shared_u32(at + (uint32_t)(j * kChannels * 4), __float_as_uint(v[j]));
              st_shared_u32(at + (uint32_t)((j + 1) * kChannels * 4), __float_as_uint(v[j + 1]));
            } else {
              const uint32_t h = pack2<T>(v[j], v[j + 1]);
              st_shared_u16(at + (uint32_t)(j * kChannels * 2), (uint16_t)h);
              st_shared_u16(at + (uint32_t)((j + 1) * kChannels * 2), (uint16_t)(h >> 16));
            }
          }
          fence_proxy_async_shared();
          named_bar_sync(bar_id, 128);
          if (issuer) {
            if (tc < p.m && c0 < p.n) tma_store_2d(&tmap_d, buf, c0, tc);
            bulk_commit_group();
          }
          ++chunk_no;
        } else if (ch_ok) {
          store_column<T, CW>(static_cast<uint8_t*>(p.d) + ((int64_t)tc * p.ldd + ch) * (int64_t)sizeof(T),
                              p.ldd * (int64_t)sizeof(T), v, p.m - tc);
        }
      }
      if (++acc == p.num_acc) { acc = 0; acc_phase ^= 1u; }
    }
    if (issuer && p.c_staged) {
      // Chunks fetched but not used (only after an abort) must land before the CTA exits.
      for (uint32_t x = chunk_no; x < c_no; ++x) drain_wait(c_full + 8u * (x % c_bufs), (x / c_bufs) & 1u, 100000000ull);
    }
    if (issuer && p.tma_store) bulk_wait_group<0>();
    }
  }

  // ------------------------------------------------------------ split-K sum and teardown
  __syncwarp();
  tc_fence_before();
  if (split) {
    cluster_arrive();
    cluster_wait();
    if (warp >= 2 && warp < 6) {
      // CTA `rank` finishes its share of the tokens: a warp takes a token, a lane four channels.
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
      // S peers and U tokens: 16 loads in flight per lane (a fused call has at most 2 tokens for a warp).
      auto finish_tokens = [&](auto s_c) {
        constexpr int S = decltype(s_c)::value, U = FUSE ? 2 : 16 / S;
        const int j_end = min((int)(rank + 1) * per, p.m - t0);
        for (int j0 = (int)rank * per + (int)warp - 2; j0 < j_end; j0 += 4 * U) {
          uint4 part[U][S];
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < S; ++s) {
              const int j = min(j0 + 4 * u, j_end - 1);
              part[u][s] = ld_shared_cluster_v4(mapa_shared(base + (uint32_t)((j * kChannels + 4 * (int)lane) * 4), (uint32_t)s));
            }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int t = t0 + j0 + 4 * u;
            if (j0 + 4 * u >= j_end) continue;
            uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S; ++s) {
              sum[0] += part[u][s].x; sum[1] += part[u][s].y; sum[2] += part[u][s].z; sum[3] += part[u][s].w;
            }
            const float sa = FUSE ? tok_rows[FUSE ? t : 0].scale : (p.sa ? p.sa[t] : 1.f);
            T* const d = static_cast<T*>(p.d) + (int64_t)t * p.ldd + ch0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (ch0 + e >= p.n) continue;
              float v = finish_large((int32_t)sum[e], sa, sb[e], bias[e]);
              if (p.drop.on) v = drop_keeps(p.drop, key, drop_index(p.drop, t, ch0 + e)) ? v * p.drop.grow : 0.f;
              if (p.c) v += to_f32(static_cast<const T*>(p.c)[(int64_t)t * p.ldc + ch0 + e]);
              d[e] = from_f32<T>(v);
            }
          }
        }
      };
      if (p.split == 2) finish_tokens(IntC<2>{});
      else if (p.split == 4) finish_tokens(IntC<4>{});
      else finish_tokens(IntC<8>{});
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
    if (a->c && !in_place_or_apart(a->c, a->ldc, a->d, a->ldd, a->m, a->n, (int64_t)e)) FAIL("C must be D or lie apart from it");
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

// Fused form: CTAs that share a tile of 128 channels.  One SM pulls some 75 of HBM's
// 6500 bytes per ns, so 64 to 128 CTAs stream at full rate; more than one wave of them costs more than it gives.
int fused_split(int64_t tiles, int64_t kb) {
  int s = 1;
  while (s < 4 && tiles * s * 2 <= 128 && kb >= 2 * s * 16) s *= 2;
  return s;
}

// Tile and split with the least estimated time, in SM cycles.  A K atom costs a CTA
// what its tensor core needs (2 BN cycles at 8192 int8 multiply-adds a cycle; a pair
// halves the tokens' rows but not this) or the bytes that it has to pull
// from L2 at some 64 a cycle, whichever is more; all of them cannot beat HBM (3400 bytes a cycle); the last
// tile's epilogue follows, 11 cycles a token.  A split of K over up to 8 CTAs (one wave; the GPU
// holds few clusters of 8 at a time) adds the exchange of the partial tiles.  Measured over all
// candidates of 30 problems of 14 to 4096 tokens, the choice is within 3 % of the best in 25
// (512 x 8192 x 8192: pairs of 256 tokens 28.6 us, of 128 32.2, single CTAs of 128 38.4, of 64 51.3;
// 496 x 965 x 21956: 128-token tiles in 4 parts 18.5, in 2 parts 23.7).  Farthest off is
// 64 x 4096 x 4096: 8.8 us in 2 parts, 32-token tiles whole 7.3.
void choose(const Int8GemmArgs* a, int num_sms, int& cg, int& bn, int& split) {
  static const int kTiles[6][2] = {{1, 16}, {1, 32}, {1, 64}, {1, 128}, {2, 128}, {2, 256}};
  const int64_t kb = (a->k + kAtom - 1) / kAtom;
  const int64_t hbm = (a->n + a->m) * a->k / 3400;
  int64_t best = INT64_MAX;
  int best_cg = cg ? cg : 1, best_bn = bn ? bn : 128, best_split = split ? split : 1;
  for (const auto& tile : kTiles) {
    const int g = tile[0], w = tile[1];
    if ((cg && g != cg) || (bn && w != bn)) continue;
    const int64_t tiles = ((a->n + kChannels * g - 1) / (kChannels * g)) * ((a->m + w - 1) / w);
    const int64_t tensor = 2 * w, load = (kChannels * kAtom + (int64_t)w / g * kAtom) / 64;
    const int64_t atom = tensor > load ? tensor : load, slots = num_sms / g;
    for (int s = 1; s <= (g == 1 ? kMaxSplit : 1); s *= 2) {
      if (split ? s != split : s > 1 && (tiles * s > (s == 8 ? 64 : 128) || kb < 8 * s)) continue;
      const int64_t waves = s > 1 ? 1 : (tiles + slots - 1) / slots, main = waves * ((kb + s - 1) / s) * atom;
      const int64_t time = (main > hbm ? main : hbm) + 11 * w + (s > 1 ? 5000 : 0);
      if (time < best) { best = time; best_cg = g; best_bn = w; best_split = s; }
    }
  }
  cg = best_cg;
  bn = best_bn;
  split = best_split;
}

// `fused`: the fused form of the linear layer is wanted (the caller has checked that it applies).
int resolve(const Int8GemmArgs* a, bool fused, Resolved& r) {
  memset(&r, 0, sizeof(r));
  const int rc = check(a, !fused, r);
  if (rc != GEMM_OK) return rc;
  r.num_sms = sm_count();
  r.cg = a->cta_group; r.bn = a->tile_n; r.split = a->split_k;
  if (fused) { r.cg = 1; r.bn = kFusedBN; r.split = fused_split((a->n + kChannels - 1) / kChannels, (a->k + kAtom - 1) / kAtom); }
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
  p.raster = p.num_cb < 2 ? 1 : 2;      // 16384 x 8192 x 8192: 760 us, 821 with 4, 808 with 8
  p.a_bytes = kChannels * kAtom;
  p.stage_bytes = p.a_bytes + (fused ? 0u : (uint32_t)(r.bn / r.cg) * kAtom);
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
  p.tma_store = r.split == 1 && a->m > 0 && rows_16b(a->d, a->ldd, e) && (a->n * e) % 16 == 0 ? 1 : 0;
  p.stg_bufs = p.tma_store ? 2 : 0;
  p.c_staged = p.tma_store && a->c && rows_16b(a->c, a->ldc, e) ? 1 : 0;
  p.c_bufs = e == 4 ? 3 : kCBufs;
  if (p.c_staged) p.stg_bufs = p.c_bufs;
  // A second epilogue group where the main loop is too short to hide one (4096 x 4096 x 1024: 18.8 us
  // with two, 22.4 with one; with bias, dropout and residual 43 and 50); its staging buffers cost
  // the ring a stage, which long main loops need.
  p.groups = r.cg == 2 && p.num_kb < (p.drop.on || p.c ? 40 : 20) ? 2 : 1;
  const int kb_cta = (p.num_kb + r.split - 1) / r.split;
  const int64_t tok_bytes = fused ? (int64_t)kb_cta * kTokAtom + kTokAtom : 0;
  const int64_t fixed = 1024 + kBarrierBytes + (int64_t)p.groups * p.stg_bufs * p.stg_bytes + p.groups * 4 * r.bn * 4 + tok_bytes + kStaticSmem;
  r.max_stages = (int)((kSmemLimit - fixed) / p.stage_bytes);
  if (r.max_stages > 12) r.max_stages = 12;
  r.stages = r.max_stages;
  if (r.split > 1) {
    if (r.stages > kb_cta) r.stages = kb_cta;
    while ((int64_t)r.stages * p.stage_bytes < (int64_t)r.bn * kChannels * 4) ++r.stages;   // the partial tile lies over the ring
  }
  p.stages = r.stages;
  p.bars_offset = (uint32_t)r.stages * p.stage_bytes;
  p.tok_offset = p.bars_offset + kBarrierBytes;
  p.stg_offset = p.tok_offset + (uint32_t)tok_bytes;
  p.k = (int32_t)a->k;
  p.sa_offset = p.stg_offset + (uint32_t)(p.groups * p.stg_bufs) * p.stg_bytes;
  r.smem_bytes = 1024 + (int64_t)p.sa_offset + p.groups * 4 * r.bn * 4;
  if (r.smem_bytes < kMinSmemPerCta) r.smem_bytes = kMinSmemPerCta;
  p.status = a->status;
  p.timeout_ns = (uint64_t)(a->timeout_ms ? a->timeout_ms : 4000u) * 1000000ull;
  p.flags = a->flags;
  const int64_t slots = r.split > 1 ? p.num_units : (r.num_sms / r.cg < p.num_units ? r.num_sms / r.cg : p.num_units);
  r.grid = (int)(slots * (r.split > 1 ? r.split : r.cg));
  return GEMM_OK;
}
#undef FAIL
#undef BAD

using KernelFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Int8Params);

template <typename T>
KernelFn pick(int cg, int bn, bool fused) {
  if (fused) return int8_gemm_kernel<1, kFusedBN, T, true>;
  if (cg == 1) {
    switch (bn) {
      case 16: return int8_gemm_kernel<1, 16, T, false>;
      case 32: return int8_gemm_kernel<1, 32, T, false>;
      case 64: return int8_gemm_kernel<1, 64, T, false>;
      default: return int8_gemm_kernel<1, 128, T, false>;
    }
  }
  return bn == 128 ? int8_gemm_kernel<2, 128, T, false> : int8_gemm_kernel<2, 256, T, false>;
}

std::mutex g_attr_mu;
struct AttrSet { KernelFn fn; int dev; };
AttrSet g_attr_set[512];
int g_attr_n = 0;

bool ensure_smem_attr(KernelFn fn, int dev, int bytes) {
  std::lock_guard<std::mutex> lock(g_attr_mu);
  for (int i = 0; i < g_attr_n; ++i)
    if (g_attr_set[i].fn == fn && g_attr_set[i].dev == dev) return true;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (g_attr_n < 512) g_attr_set[g_attr_n++] = {fn, dev};
  return true;
}

struct Tokens {        // floating tokens of the fused form
  const void* x;
  int64_t ldx;
};

// A product that is ready to be launched: nothing can refuse it any more.
struct Prepared {
  Resolved r;
  CUtensorMap tw, tt, td, tc;
  KernelFn fn;
  int threads;
};

// The device of D is current.
int prepare_product(const Int8GemmArgs& a, const Tokens* tokens, int dev, Prepared& q) {
  Resolved& r = q.r;
  const int rc = resolve(&a, tokens != nullptr, r);
  if (rc != GEMM_OK) return rc;
  if (!get_encode()) return GEMM_ERR_LAUNCH;
  memset(&q.tt, 0, sizeof(q.tt));
  memset(&q.td, 0, sizeof(q.td));
  memset(&q.tc, 0, sizeof(q.tc));
  if (!encode_2d(&q.tw, a.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)a.k, (uint64_t)a.n, (uint64_t)a.ldb, kAtom, kChannels, 128))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (tokens) {
    r.p.x = tokens->x;
    r.p.ldx = tokens->ldx;
    r.p.x_wide = rows_16b(tokens->x, tokens->ldx, type_bytes(a.d_type)) ? 1 : 0;
  } else if (!encode_2d(&q.tt, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)a.k, (uint64_t)a.m, (uint64_t)a.lda, kAtom,
                        (uint32_t)(r.bn / r.cg), 128)) {
    return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  if (r.p.tma_store) {
    const CUtensorMapDataType t = a.d_type == GEMM_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : a.d_type == GEMM_TYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    const uint32_t tokens_box = (uint32_t)(r.bn < 32 ? r.bn : 32);
    if (!encode_2d(&q.td, a.d, t, (uint64_t)a.n, (uint64_t)a.m, (uint64_t)(a.ldd * type_bytes(a.d_type)), kChannels, tokens_box, 0))
      return GEMM_ERR_CANNOT_IMPLEMENT;
    if (r.p.c_staged &&
        !encode_2d(&q.tc, a.c, t, (uint64_t)a.n, (uint64_t)a.m, (uint64_t)(a.ldc * type_bytes(a.d_type)), kChannels, tokens_box, 0))
      return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  q.fn = a.d_type == GEMM_TYPE_BF16 ? pick<__nv_bfloat16>(r.cg, r.bn, tokens != nullptr)
       : a.d_type == GEMM_TYPE_FP16 ? pick<__half>(r.cg, r.bn, tokens != nullptr) : pick<float>(r.cg, r.bn, tokens != nullptr);
  q.threads = tokens ? threads_for(1, true) : 64 + 128 * r.p.groups;
  return ensure_smem_attr(q.fn, dev, tokens ? kSmemLimit - kStaticSmem : kSmemLimit) ? GEMM_OK : GEMM_ERR_LAUNCH;
}

int launch_prepared(const Prepared& q, cudaStream_t st) {
  const Resolved& r = q.r;
  if (launch_overlapped(q.fn, dim3((unsigned)r.grid), dim3((unsigned)q.threads), (size_t)r.smem_bytes,
                        r.split > 1 ? r.split : r.cg, st, q.tw, q.tt, q.td, q.tc, r.p) != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}

// Few tokens, no knob set and X of D's type: one launch.  Every CTA then quantises
// the tokens for itself, which costs more than the launch it saves beyond some
// 16384 of their elements: 8192 x 8192, 1 token 14.5 us against 17.2 in two
// launches, 4 tokens 18.0 against 17.2.  A D that lies over the tokens (the layer's result
// replaces them) needs two launches, the tokens being quantised before the first store.
bool use_fused(const Int8GemmArgs& a, const void* x, int32_t x_type, int64_t ldx) {
  return a.m <= kFusedTokens && a.m * a.k <= kFusedElems && x_type == a.d_type && !a.tile_n && !a.cta_group && !a.split_k &&
         !a.flags && (a.m < 1 || !rows_meet(x, ldx * type_bytes(x_type), a.k * type_bytes(x_type), a.d,
                                            a.ldd * type_bytes(x_type), a.n * type_bytes(x_type), a.m));
}

}  // namespace

extern "C" int gemm_sm100a_int8_query(const Int8GemmArgs* args, GemmInfo* info) {
  Resolved r;
  const int rc = resolve(args, false, r);
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
  PointerDeviceGuard guard(args->d);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  Prepared q;
  const int rp = prepare_product(*args, nullptr, guard.dev, q);
  return rp != GEMM_OK ? rp : launch_prepared(q, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int gemm_sm100a_int8_linear(const Int8GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream) {
  Resolved r;
  memset(&r, 0, sizeof(r));
  const bool few = args && args->struct_size == sizeof(Int8GemmArgs) && use_fused(*args, x, x_type, ldx);
  const int rc = check(args, !few, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  if (!type_ok(x_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!x || (!few && !args->scale_a)) return GEMM_ERR_BAD_ARGS;
  if (ldx < args->k || reinterpret_cast<uintptr_t>(x) % type_bytes(x_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(args->d);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  // The product is prepared before the tokens are quantised: a refused call launches nothing.
  const Tokens tokens = {x, ldx};
  Prepared p;
  const int rp = prepare_product(*args, few ? &tokens : nullptr, guard.dev, p);
  if (rp != GEMM_OK) return rp;
  if (!few) {
    Int8QuantArgs q;
    memset(&q, 0, sizeof(q));
    q.struct_size = sizeof(q);
    q.x_type = x_type; q.rows = args->m; q.cols = args->k; q.x = x; q.ldx = ldx;
    q.q = const_cast<void*>(args->a); q.ldq = args->lda; q.scale = const_cast<float*>(args->scale_a);
    const int rq = gemm_sm100a_quantize_int8(&q, stream);
    if (rq != GEMM_OK) return rq;
  }
  return launch_prepared(p, st);
}
