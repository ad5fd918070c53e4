// fp4_gemm.cu -- product of 4-bit operands with block and row scales:
//   D[i][j] = C[i][j] + ra[i] * rb[j] * sum_k A[i][k] B[j][k] + bias[j]
//
// tcgen05.mma kind::mxf4nvf4 (blocks of 16, e4m3 scales) or kind::mxf4 (blocks of 32, powers of two), fp32
// accumulators in TMEM.  Channels (rows of B) lie on the MMA's M side, tokens (rows of A) on its N side, as in
// the int8 product: a weight tile is always a full 128 rows however few tokens there are, a thread keeps its
// channel's scale and bias in registers, and a warp's 32 lanes write 32 consecutive elements of a row of D.
//
// Warp 0 loads 128-byte K atoms (256 elements) and their scale tiles into a ring, warp 1 copies
// the scales to tensor memory (tcgen05.cp) and issues the MMAs, warps 2..5 run the epilogue (one TMEM lane quadrant
// each; in a pair warps 6..9 take every other chunk).
//   whole-K form   persistent CTAs (CTA pairs for large problems), two
//                  accumulators, so a tile's epilogue overlaps the next mainloop.  Two of 256
//                  tokens and two atoms' scales do not fit in tensor memory: their positions overlap by 96 columns, which
//                  the epilogue reads first.
//   split-K form   for few tiles: the CTAs of a cluster share one tile's K and
//                  add their fp32 partial tiles in the order of their ranks through distributed shared
//                  memory; no workspace.
//   fused form     for a linear layer of at most 8 tokens, in one launch: while the
//                  ring fills with weights, 12 warps find the tokens' maxima and
//                  quantise the CTA's part of them straight into the swizzled
//                  operand and its scale tiles, which stay in shared memory for all of its tiles.
//
// Measured on B200: 8192 x 28672 x 8192 in 748 to 790 us at the clock that the power cap leaves (4.9 to 5.1
// PFLOP/s), 4096 x 8192 x 8192 in 106 (5.2); 48 x 28672 x 8192 in 26.5, its 132 MB at 5 of the 6.55 TB/s that a copy
// reaches; one token x 8192 x 8192 in 10.0 in one launch, of which some 4 are launch, first loads and last stores.
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
#include "fp4_common.cuh"
#include "row_vec.cuh"
#include "tensor_map.cuh"

using namespace sm100;
using namespace int8op;

namespace {

constexpr int kFusedTokens = 8;         // most tokens of the fused form: one 8-row group of the swizzle
constexpr int kFusedBN = 16;            // its MMA N, the smallest there is for 128 channels
constexpr int kStageWarps = 12;         // warps of the fused form that quantise tokens (the epilogue's four among them)
constexpr int kFusedElems = 16384;      // most tokens x K (in whole atoms) of the fused form: at most 96 KB of shared memory
constexpr int kMaxGroups = 2;           // epilogue groups of a CTA pair's kernel (four warps each)
constexpr int kOverlap = 96;            // columns that the two positions of a 256-token accumulator share: three chunks of the epilogue
constexpr int kTmemCols = 512;          // all of it: one CTA per SM
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
constexpr int kScaleBars = 4;
constexpr int kCBufs = 4;               // most staging buffers of an epilogue group that reads C by TMA:
                                        // all but two hold chunks of C on their way
constexpr int kAtom = 128;              // bytes of one swizzled K atom
constexpr int kAtomK = fp4op::kAtomK;   // its K elements
constexpr uint32_t kTokAtom = 8 * kAtom;  // fused form: bytes of one K atom of the tokens
constexpr uint32_t kTokTile = 128;      // fused form: bytes of one scale tile of 8 tokens x 4 scales (rows 16 bytes apart)
__host__ __device__ constexpr int tiles_per_atom(int block) { return kAtomK / 4 / block; }
constexpr int kChannels = 128;          // channels per CTA
constexpr int kMaxStages4 = 12;         // most stages of a ring (the barriers have room for kMaxStages)
// A copy of scales to tensor memory is ordered behind the MMAs that read what it overwrites by nothing but their commit.  They have as
// many slots as there are stages, whose loads have waited for that commit: then nothing more has to be waited for.  The 256-token
// tile has room for two slots (blocks of 16) or four (blocks of 32), each with a barrier that its issuer waits for (4096 x 8192 x 8192,
// blocks of 16: 105.8 us; 103.3 with one slot that nothing guarded, 117 with four slots of half an atom).
__host__ __device__ constexpr int slot_columns(int bn, int block) { return tiles_per_atom(block) * 4 * (1 + (bn + 127) / 128); }
__host__ __device__ constexpr int first_slot(int bn) { return bn == 256 ? 2 * bn - kOverlap : 2 * bn; }           // behind the accumulators
__host__ __device__ constexpr int scale_slots(int bn, int block) {
  const int n = (kTmemCols - first_slot(bn)) / slot_columns(bn, block);
  return n < kMaxStages4 ? n : kMaxStages4;
}
constexpr int kMaxSplit = 8;            // CTAs that may share a tile's K (portable cluster size)

template <int V>
struct IntC { static constexpr int value = V; };

struct Fp4Params {
  void* d; int64_t ldd;
  const void* c; int64_t ldc;
  const float* sa;
  const float* sb;
  const void* bias;
  int32_t bias_type;
  int32_t m, n;
  const uint8_t* ts;                    // scale tiles of the tokens and of the channels
  const uint8_t* ws;
  int64_t tiles;                        // scale tiles along a row
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
  int32_t num_acc;
  int32_t raster;                       // channel blocks per raster group
  uint32_t idesc;
  int32_t* status;
  uint64_t timeout_ns;
  uint32_t flags;
  const void* x; int64_t ldx;           // fused form: tokens before quantisation
  int32_t k;
  uint32_t tok_offset, tok_tiles;       // fused form: quantised tokens, kTokAtom bytes per K atom, and their scale tiles
};

// Block-scaled kinds: [4,6) B scale id, [7,10) A format (1 = E2M1), [10,12) B format, [17,23) N >> 3, [23] scale
// type (0 = UE4M3, 1 = UE8M0), [24,29) M >> 4, [29,31) A scale id.
__host__ constexpr uint32_t make_idesc(int mma_m, int mma_n, int block) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(mma_n >> 3) << 17) | (block == 32 ? 1u << 23 : 0u) | ((uint32_t)(mma_m >> 4) << 24);
}
// Scale ids of the second MMA of a word of four scales (two to an MMA).
constexpr uint32_t kUpperScales = (2u << 4) | (2u << 29);

// One output from its sum.
__device__ __forceinline__ float finish(float acc, float sa, float sb, float bias) { return fmaf(acc * sa, sb, bias); }
// The sum (below 2^40) times a larger scale than this might leave the range of fp32 where the output does not; the
// channel's scale then comes first.
constexpr float kLargeScale = 0x1p84f;
__device__ __forceinline__ bool is_large(float sa) { return fabsf(sa) > kLargeScale; }
__device__ __forceinline__ float finish_large(float acc, float sa, float sb, float bias) {
  const bool large = is_large(sa);
  return finish(acc, large ? sb : sa, large ? sa : sb, bias);
}

__device__ __forceinline__ void tile_coords(int u, const Fp4Params& p, int& cb, int& tb) {
  const int per_group = p.raster * p.num_tb;
  const int g = u / per_group;
  const int first = g * p.raster;
  const int rows = min(p.num_cb - first, p.raster);
  const int r = u - g * per_group;
  cb = first + r % rows;
  tb = r / rows;
}

// Fused form: all staging warps, `tid` in [0, 32 * kStageWarps).  Each thread keeps up to three units of the
// tokens in registers, so x is read once; atoms [kb_begin, kb_end) of the quantised rows go to `tok`, 128-byte
// rows in the 128-byte swizzle, their scales to `tiles`, their row scales to `sa_s`.
// Rows from m on stay undefined: those accumulator columns are not read.  (Rows 8 to 15 of the MMA's
// operand are the next K atom's, after the last one the 1 KB behind it; rows 8 to 31 of a scale tile the next three
// tiles', after the last one the 384 bytes behind it.)
template <typename X, int BLOCK>
__device__ __forceinline__ void stage_tokens(const Fp4Params& p, uint32_t tok, uint32_t tiles, uint32_t sa_s, uint32_t* top,
                                             int kb_begin, int kb_end, int tid) {
  constexpr int N = 32 * kStageWarps, PER = (kFusedElems / 16 + N - 1) / N;
  const X* const x = static_cast<const X*>(p.x);
  const int width = p.num_kb * (kAtomK / 16);       // units of a token: whole atoms, so 16 lanes hold one token's
  const int total = p.m * width;
  if (tid < kFusedTokens) top[tid] = 0u;
  __syncwarp();
  named_bar_sync(2, N);
  rowvec::Unit<X> v[PER];
  uint32_t tops[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int u = i * N + tid, t = u / width, e = (u - t * width) * 16;
    v[i] = rowvec::load_unit<X, rowvec::kKeep>(x + (u < total ? t * p.ldx + e : 0), u < total ? p.k - e : 0);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    uint32_t m = tops[i] = rowvec::magnitude(v[i]);
#pragma unroll
    for (int o = 1; o < 16; o *= 2) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const int u = i * N + tid;
    if (u < total && (tid & 15) == 0) atomicMax(&top[u / width], m);
  }
  __syncwarp();
  named_bar_sync(2, N);
  // Each of the epilogue's warps writes them for itself (the same values).
  const int who = tid & 31;
  if (tid < 128 && who < p.m) st_shared_u32(sa_s + 4u * who, __float_as_uint(fp4op::row_scale(top[who]).scale));
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int u = i * N + tid, t = min(u / width, kFusedTokens - 1), unit = u - u / width * width;
    const fp4op::RowScale s = fp4op::row_scale(top[t]);
    const bool far = s.far();
    float y[16], most = __uint_as_float(tops[i]);
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = v[i].get(j);
    if (far) fp4op::bring_near(y, most, s);
    uint32_t q[2];
    const uint32_t code = fp4op::quantize_unit<BLOCK>(y, most, far ? 1.f : s.up, far ? 1.f : s.scale, q);
    constexpr int STEP = BLOCK / 16;
    uint32_t w = code << (8 * ((tid / STEP) & 3));
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, STEP);
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 2 * STEP);
    const int atom = unit / 16 - kb_begin, in = unit & 15;
    if (u >= total || atom < 0 || atom >= kb_end - kb_begin) continue;
    st_shared_v2(tok + (uint32_t)atom * kTokAtom + (uint32_t)t * 128u + (((uint32_t)(in >> 1) ^ (uint32_t)t) << 4) + 8u * (in & 1), q[0], q[1]);
    if (in % (4 * STEP) == 0) st_shared_u32(tiles + (uint32_t)(atom * tiles_per_atom(BLOCK) + in / (4 * STEP)) * kTokTile + (uint32_t)t * 16u, w);
  }
}

// One element of a staged chunk.
template <typename T>
__device__ __forceinline__ float staged(uint32_t addr) {
  const uint16_t h = ld_shared_u16(addr);
  T v;
  __builtin_memcpy(&v, &h, 2);
  return to_f32(v);
}

// A thread's column of a chunk, `tokens` rows of D from `d`, `step` bytes apart: for
// a D that TMA cannot store.  With one warp per scheduler every instruction counts, hence the running
// pointer and the paired conversions.
template <typename T, int CW>
__device__ __forceinline__ void store_column(uint8_t* d, int64_t step, const float (&v)[CW], int tokens) {
#pragma unroll
  for (int j = 0; j < CW; j += 2) {
    uint8_t* const d1 = d + step;
    const uint32_t h = pack2<T>(v[j], v[j + 1]);
    if (j < tokens) *reinterpret_cast<uint16_t*>(d) = (uint16_t)h;
    if (j + 1 < tokens) *reinterpret_cast<uint16_t*>(d1) = (uint16_t)(h >> 16);
    d = d1 + step;
  }
}

template <int CG, int BN, int BLOCK, typename T, bool FUSE>
__global__ void __launch_bounds__(threads_for(CG, FUSE), 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w,   // weights: channels x K
                 const __grid_constant__ CUtensorMap tmap_t,   // tokens x K
                 const __grid_constant__ CUtensorMap tmap_d,   // D, for the staged epilogue
                 const __grid_constant__ CUtensorMap tmap_c,   // C, where it is staged too
                 const __grid_constant__ CUtensorMap tmap_ws,  // scale tiles of the channels and of the tokens (pairs)
                 const __grid_constant__ CUtensorMap tmap_ts,
                 const __grid_constant__ Fp4Params p) {
  constexpr int TROWS = BN / CG;                    // token rows each CTA of a pair loads
  constexpr int CW = BN < 32 ? BN : 32;             // tokens per epilogue chunk
  constexpr int NCH = BN / CW;
  constexpr int NSF = tiles_per_atom(BLOCK);        // scale tiles of a K atom
  constexpr int TB = (BN + 127) / 128;              // row blocks of 128 tokens
  constexpr int OV = BN == 256 ? kOverlap : 0;      // columns that the accumulator's two positions share
  constexpr uint32_t SF0 = first_slot(BN), SF_COLS = slot_columns(BN, BLOCK), SF_SLOTS = scale_slots(BN, BLOCK);
  constexpr bool SF_WAIT = BN == 256;
  static_assert(!SF_WAIT || (CG == 2 && SF_SLOTS >= 2 && SF_SLOTS <= kScaleBars), "scales of two atoms fit behind the accumulators");

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
  const uint32_t scale_bar = lost_flag0 + 4u * kMaxGroups;        // [kScaleBars]: the MMAs have read a slot's scales
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
    if constexpr (CG == 2) {
      prefetch_tmap(&tmap_ws);
      prefetch_tmap(&tmap_ts);
    }
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
    for (int b = 0; b < kScaleBars; ++b) mbar_init(scale_bar + 8u * b, 1);
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
    tmem_alloc<CG>(tmem_slot, (uint32_t)kTmemCols);
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
              // The pair's MMA reads every token's scale from each CTA's own tensor memory.
              const uint32_t sf_dst = t_dst + (uint32_t)(TROWS * kAtom);
              tma_load_3d_pair(sf_dst, &tmap_ws, target, 0, kb * NSF, c0 / 128, policy, issue);
              tma_load_3d_pair(sf_dst + NSF * 512u, &tmap_ts, target, 0, kb * NSF, tb * TB, policy, issue);
            } else {
              tma_load_2d(w_dst, &tmap_w, target, kb * kAtom, c0, policy, issue);
              const uint32_t sf_dst = FUSE ? t_dst : t_dst + (uint32_t)(TROWS * kAtom);
              bulk_load(sf_dst, p.ws + ((int64_t)cb * p.tiles + kb * NSF) * 512, NSF * 512u, target, policy, issue);
              if constexpr (!FUSE) {
                tma_load_2d(t_dst, &tmap_t, target, kb * kAtom, t0, policy, issue);
                bulk_load(sf_dst + NSF * 512u, p.ts + ((int64_t)tb * p.tiles + kb * NSF) * 512, NSF * 512u, target, policy, issue);
              }
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
      uint32_t phase = 0, acc_phase = 0, pos = 0, slot = 0, slot_phase = 0;
      bool ok = true, issued = false;
      if constexpr (FUSE) {
        const bool wt = wait_bar<false>(tok_bar, 0, ctl, ROLE_MMA, 0x90u);
        ok = __all_sync(0xffffffffu, wt);
      }
      for (int u = slot0; u < p.num_units && ok; u += slots) {
        const bool wt = wait_bar<CG == 2>(tempty_bar + 8u * acc, acc_phase ^ 1u, ctl, ROLE_MMA, 0x80u | acc);
        if (!__all_sync(0xffffffffu, wt)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (OV ? pos * (uint32_t)(BN - OV) : (uint32_t)(acc * BN));
        pos ^= 1u;
        bool ready = false;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          const bool w = ready || wait_bar<CG == 2>(full_bar + 8u * stage, phase, ctl, ROLE_MMA, stage);
          if (!w) { ok = false; break; }
          tc_fence_after();
          const uint32_t w_src = base + (uint32_t)stage * p.stage_bytes;
          const uint32_t t_src = w_src + p.a_bytes;
          const uint32_t ws_src = FUSE ? t_src : t_src + (uint32_t)(TROWS * kAtom);
          const uint32_t ts_src = FUSE ? base + p.tok_tiles + (uint32_t)((kb - kb_begin) * NSF) * kTokTile : ws_src + NSF * 512u;
          const uint64_t wd = sw128_kmajor_desc(w_src);
          const uint64_t td = sw128_kmajor_desc(FUSE ? base + p.tok_offset + (uint32_t)(kb - kb_begin) * kTokAtom : t_src);
          if constexpr (SF_WAIT) {
            if (!wait_bar<false>(scale_bar + 8u * slot, slot_phase ^ 1u, ctl, ROLE_MMA, 0xA0u | slot)) { ok = false; break; }
            tc_fence_after();
          }
          if (CG == 1 || issue) {
            const uint32_t ws_t = tmem_base + SF0 + slot * SF_COLS, ts_t = ws_t + NSF * 4u;
            const uint64_t ws_desc = plain_desc(ws_src), ts_desc = plain_desc(ts_src);      // (in units of 16 bytes)
#pragma unroll
            for (int q = 0; q < NSF; ++q) {
              tmem_cp_32x128b_warpx4<CG>(ws_t + 4u * q, ws_desc + 32u * q, issue);
#pragma unroll
              for (int b = 0; b < TB; ++b)
                tmem_cp_32x128b_warpx4<CG>(ts_t + (uint32_t)(q * TB + b) * 4u, ts_desc + (FUSE ? kTokTile / 16u * q : (uint32_t)(b * NSF + q) * 32u), issue);
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint32_t acc_on = (kb != kb_begin || kk) ? 1u : 0u;
              if constexpr (BLOCK == 16)
                mma_nvf4<CG>(d_tmem, wd + 2u * kk, td + 2u * kk, p.idesc, ws_t + 4u * kk, ts_t + 4u * TB * kk, acc_on, issue);
              else
                mma_mxf4<CG>(d_tmem, wd + 2u * kk, td + 2u * kk, p.idesc | (kk & 1 ? kUpperScales : 0u), ws_t + 4u * (kk / 2),
                             ts_t + 4u * TB * (kk / 2), acc_on, issue);
            }
            if constexpr (SF_WAIT) mma_commit_pair(scale_bar + 8u * slot, 0x1, issue);
            if constexpr (CG == 2) mma_commit_pair(empty_bar + 8u * stage, 0x3, issue);
            else mma_commit(empty_bar + 8u * stage, issue);
          }
          issued = true;
          if (++slot == SF_SLOTS) { slot = 0; slot_phase ^= 1u; }
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
      stage_tokens<T, BLOCK>(p, base + p.tok_offset, base + p.tok_tiles, base + p.sa_offset, tok_top, kb_begin, kb_end, (int)threadIdx.x - 64);
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
    uint32_t chunk_no = 0;
    // C staged: chunk x of this group (over all its tiles) goes through buffer x % c_bufs, is
    // replaced there by D, element by element in the same thread, and stored from it.  One
    // thread fetches c_bufs - 2 chunks ahead, also across tiles.
    const uint32_t c_bufs = (uint32_t)p.c_bufs;
    int c_u = slot0, c_i = (int)grp;
    uint32_t c_no = 0, c_pos = 0;
    const uint64_t c_policy = policy_evict_normal();
    // The i-th chunk of a tile: those that overlap the accumulator's other position first.
    auto chunk_at = [](int i, uint32_t pos) { return OV && pos == 0 ? (i + NCH - OV / CW) % NCH : i; };
    auto fetch_c = [&]() {
      if (c_u >= p.num_units) return;
      int cb, tb;
      tile_coords(c_u, p, cb, tb);
      const uint32_t buf = c_no % c_bufs;
      mbar_arrive_expect_tx(c_full + 8u * buf, p.stg_bytes);
      tma_load_2d(stg + buf * p.stg_bytes, &tmap_c, c_full + 8u * buf,
                  (cb * CG + (int)(CG == 2 ? rank : 0u)) * kChannels, tb * BN + chunk_at(c_i, c_pos) * CW, c_policy);
      ++c_no;
      if ((c_i += groups) >= NCH) { c_i = (int)grp; c_u += slots; c_pos ^= 1u; }
    };
    if (p.c_staged && issuer) {
      for (uint32_t b = 2; b < c_bufs; ++b) fetch_c();
    }
    int acc = 0;
    uint32_t acc_phase = 0, pos = 0;
    for (int u = slot0; u < p.num_units; u += slots, pos ^= 1u) {
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
      }
      // (Fused form: the staging warps' scales are in place before any sum is.)
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
      if constexpr (FUSE) large = (int)lane < p.m && is_large(__uint_as_float(ld_shared_u32(sa_s + 4u * (lane & (kFusedTokens - 1)))));
      large = __any_sync(0xFFFFFFFFu, large);
      const uint32_t t_row = tmem_base + ((32u * q) << 16) + (OV ? pos * (uint32_t)(BN - OV) : (uint32_t)(acc * BN));
      if (split) {
        // This CTA's partial tile, [token][channel] fp32, over the ring: every
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
        const int at_chunk = chunk_at(i, pos);
        uint32_t r[CW];
        if constexpr (CW == 32) tmem_ld32(t_row + (uint32_t)(at_chunk * CW), r); else tmem_ld16(t_row + (uint32_t)(at_chunk * CW), r);
        tmem_ld_wait();
        if (OV ? i < OV / CW && i + groups >= OV / CW : i + groups >= NCH) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(leader_tempty + 8u * acc); else mbar_arrive(tempty_bar + 8u * acc);
          }
        }
        const int tc = t0 + at_chunk * CW;
        float v[CW];
        if (!large) {
#pragma unroll
          for (int j = 0; j < CW; j += 4) {
            const uint4 sa = ld_shared_v4(sa_s + 4u * (uint32_t)(at_chunk * CW + j));
            v[j] = finish(__uint_as_float(r[j]), __uint_as_float(sa.x), sb, bias);
            v[j + 1] = finish(__uint_as_float(r[j + 1]), __uint_as_float(sa.y), sb, bias);
            v[j + 2] = finish(__uint_as_float(r[j + 2]), __uint_as_float(sa.z), sb, bias);
            v[j + 3] = finish(__uint_as_float(r[j + 3]), __uint_as_float(sa.w), sb, bias);
          }
        } else {
#pragma unroll
          for (int j = 0; j < CW; ++j)
            v[j] = finish_large(__uint_as_float(r[j]), __uint_as_float(ld_shared_u32(sa_s + 4u * (uint32_t)(at_chunk * CW + j))), sb, bias);
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
            const uint32_t h = pack2<T>(v[j], v[j + 1]);
            st_shared_u16(at + (uint32_t)(j * kChannels * 2), (uint16_t)h);
            st_shared_u16(at + (uint32_t)((j + 1) * kChannels * 2), (uint16_t)(h >> 16));
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
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
              sum[0] += __uint_as_float(part[u][s].x); sum[1] += __uint_as_float(part[u][s].y);
              sum[2] += __uint_as_float(part[u][s].z); sum[3] += __uint_as_float(part[u][s].w);
            }
            const float sa = FUSE ? __uint_as_float(ld_shared_u32(base + p.sa_offset + 4u * (uint32_t)t)) : (p.sa ? p.sa[t] : 1.f);
            T* const d = static_cast<T*>(p.d) + (int64_t)t * p.ldd + ch0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (ch0 + e >= p.n) continue;
              float v = finish_large(sum[e], sa, sb[e], bias[e]);
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
    tmem_dealloc<CG>(tmem_base, (uint32_t)kTmemCols);
  }
}

// ----------------------------------------------------------------- host
struct Resolved {
  int cg, bn, split, stages, max_stages;
  int grid, num_sms;
  int64_t smem_bytes;
  Fp4Params p;
  char reason[128];
};

#define FAIL(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_CANNOT_IMPLEMENT; } while (0)
#define BAD(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_BAD_ARGS; } while (0)

// `tokens`: A and its scales are read or written (not by the few-token form of the linear layer).
int check(const Fp4GemmArgs* a, bool tokens, Resolved& r) {
  if (!a) BAD("null args");
  if (a->struct_size != sizeof(Fp4GemmArgs)) BAD("Fp4GemmArgs.struct_size %u != %zu", a->struct_size, sizeof(Fp4GemmArgs));
  if (a->d_type != GEMM_TYPE_BF16 && a->d_type != GEMM_TYPE_FP16) FAIL("d_type %d: the result is bf16 or fp16", a->d_type);
  if (!fp4op::block_ok(a->block)) FAIL("block %d must be 16 or 32", a->block);
  if (a->bias && !type_ok(a->bias_type)) FAIL("unknown bias_type %d", a->bias_type);
  if (a->m < 0 || a->n < 0 || a->k <= 0) FAIL("empty problem %lld x %lld x %lld", (long long)a->m, (long long)a->n, (long long)a->k);
  if (a->m > INT32_MAX / 2 || a->n > INT32_MAX / 2 || a->k > INT32_MAX / 2) FAIL("dimension too large");
  if (a->flags & ~(uint32_t)GEMM_FLAG_INJECT_STALL) FAIL("unknown flags 0x%x", a->flags);
  if (a->m > 0 && a->n > 0) {
    if ((tokens && (!a->a || !a->a_scales)) || !a->b || !a->b_scales || !a->d) BAD("null A/B/scales/D pointer");
    const uintptr_t pa = tokens ? reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->a_scales) : 0;
    const int64_t lda = tokens ? a->lda : a->ldb;
    if ((pa | reinterpret_cast<uintptr_t>(a->b) | reinterpret_cast<uintptr_t>(a->b_scales)) & 15) FAIL("A/B and their scales must be 16-byte aligned");
    if (lda < (a->k + 1) / 2 || a->ldb < (a->k + 1) / 2) FAIL("lda/ldb must be >= k / 2");
    if ((lda | a->ldb) & 15) FAIL("lda/ldb must be multiples of 16");
    const int64_t e = type_bytes(a->d_type);
    if ((reinterpret_cast<uintptr_t>(a->d) | reinterpret_cast<uintptr_t>(a->c)) % (uintptr_t)e) FAIL("D/C must be aligned to their element");
    if (a->ldd < a->n) FAIL("ldd must be >= n");
    if (a->c && a->ldc < a->n) FAIL("ldc must be >= n");
    if (a->c && !in_place_or_apart(a->c, a->ldc, a->d, a->ldd, a->m, a->n, e)) FAIL("C must be D or lie apart from it");
    if ((reinterpret_cast<uintptr_t>(a->a_row_scale) | reinterpret_cast<uintptr_t>(a->b_row_scale)) & 3) FAIL("row scales must be 4-byte aligned");
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

// Fused form: CTAs that share a tile of 128 channels.  64 to 128 CTAs stream at HBM's rate, and a part has at least 8 atoms of
// K (1 x 8192 x 8192: 10.0 us in 2 parts).
int fused_split(int64_t tiles, int64_t kb) {
  int s = 1;
  while (s < 4 && tiles * s * 2 <= 128 && kb >= 2 * s * 8) s *= 2;
  return s;
}

// Tile and split with the least estimated time, in SM cycles.  A K atom costs a CTA
// what its tensor core needs (2 BN cycles at 16384 multiply-adds a cycle; a pair
// halves the tokens' rows but not this) or the bytes that it has to pull
// from L2 at some 64 a cycle, whichever is more; all of them cannot beat HBM (3400 bytes a cycle); the last
// tile's epilogue follows, 11 cycles a token.  A split of K over up to 8 CTAs (one wave; the GPU
// holds few clusters of 8 at a time) adds the exchange of the partial tiles.  Tiles of fewer than 128 tokens
// take all tokens at once (their scales begin with a tile of 128 rows).  Over 45 problems of 16 to 400 tokens the choice is within 4 %
// of the best candidate in 37 (48 x 28672 x 8192: 26.4 us with 64 tokens, 27.5 in pairs; 64 x 1000 x 8000: 5.8 in 8 parts, 6.2 in 4,
// 8.3 in 2).  Farthest off are 192 and 256 x 4096 x 4096: 8.3 us in pairs, 7.5 with single CTAs of 128.
void choose(const Fp4GemmArgs* a, int num_sms, int& cg, int& bn, int& split) {
  static const int kTiles[6][2] = {{1, 16}, {1, 32}, {1, 64}, {1, 128}, {2, 128}, {2, 256}};
  const int64_t kb = (a->k + kAtomK - 1) / kAtomK, sf = tiles_per_atom(a->block) * 512;
  const int64_t hbm = (a->n + a->m) * kb * 144 / 3400;
  int64_t best = INT64_MAX;
  int best_cg = cg ? cg : 1, best_bn = bn ? bn : 128, best_split = split ? split : 1;
  for (const auto& tile : kTiles) {
    const int g = tile[0], w = tile[1];
    if ((cg && g != cg) || (bn && w != bn) || (w < 128 && a->m > w)) continue;
    const int64_t tiles = ((a->n + kChannels * g - 1) / (kChannels * g)) * ((a->m + w - 1) / w);
    const int64_t tensor = 2 * w, load = (kChannels * kAtom + (int64_t)w / g * kAtom + sf * (1 + (w + 127) / 128)) / 64;
    const int64_t atom = tensor > load ? tensor : load, slots = num_sms / g;
    for (int s = 1; s <= (g == 1 ? kMaxSplit : 1); s *= 2) {
      if (split ? s != split : s > 1 && (tiles * s > (s == 8 ? 64 : 128) || kb < 4 * s)) continue;
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
int resolve(const Fp4GemmArgs* a, bool fused, Resolved& r) {
  memset(&r, 0, sizeof(r));
  const int rc = check(a, !fused, r);
  if (rc != GEMM_OK) return rc;
  r.num_sms = sm_count();
  Fp4Params& p = r.p;
  p.num_kb = (int)((a->k + kAtomK - 1) / kAtomK);
  r.cg = a->cta_group; r.bn = a->tile_n; r.split = a->split_k;
  if (fused) { r.cg = 1; r.bn = kFusedBN; r.split = fused_split((a->n + kChannels - 1) / kChannels, p.num_kb); }
  choose(a, r.num_sms, r.cg, r.bn, r.split);
  if (r.cg != 1 && r.cg != 2) FAIL("cta_group must be 1 or 2");
  if (!supported(r.cg, r.bn)) FAIL("tile_n %d unsupported for cta_group %d", r.bn, r.cg);
  if (r.bn < 128 && a->m > r.bn) FAIL("tile_n %d below 128 must hold all %lld tokens", r.bn, (long long)a->m);
  if (r.split != 1 && r.split != 2 && r.split != 4 && r.split != 8) FAIL("split_k must be 1, 2, 4 or 8");
  if (r.split > 1) {
    if (r.cg != 1) FAIL("split_k needs cta_group 1");
    if (r.split > p.num_kb) FAIL("split_k %d of %d K blocks", r.split, p.num_kb);
  }
  p.split = r.split;
  p.d = a->d; p.ldd = a->ldd; p.c = a->c; p.ldc = a->ldc;
  p.sa = a->a_row_scale; p.sb = a->b_row_scale; p.bias = a->bias; p.bias_type = a->bias_type;
  p.ts = static_cast<const uint8_t*>(a->a_scales); p.ws = static_cast<const uint8_t*>(a->b_scales);
  p.tiles = fp4op::scale_tiles(a->k, a->block);
  p.m = (int32_t)a->m; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
  p.num_cb = (int)((a->n + kChannels * r.cg - 1) / (kChannels * r.cg));
  p.num_tb = (int)((a->m + r.bn - 1) / r.bn);
  if ((int64_t)p.num_cb * p.num_tb > INT32_MAX / 16) FAIL("too many tiles");
  p.num_units = p.num_cb * p.num_tb;
  p.raster = p.num_cb < 2 ? 1 : 2;
  const int sf = tiles_per_atom(a->block);
  p.a_bytes = kChannels * kAtom;
  p.stage_bytes = p.a_bytes + sf * 512u + (fused ? 0u : (uint32_t)(r.bn / r.cg) * kAtom + (uint32_t)((r.bn + 127) / 128) * sf * 512u);
  p.num_acc = r.split > 1 || r.bn == 256 ? 1 : 2;
  p.idesc = make_idesc(kChannels * r.cg, r.bn, a->block);
  // Shared memory: ring, barriers, tokens (fused form), staging (whole-K form, when D allows TMA stores), token scales.
  const int e = type_bytes(a->d_type);
  const int cw = r.bn < 32 ? r.bn : 32;
  p.stg_bytes = (uint32_t)(cw * kChannels * e);
  // (A TMA store whose row extent ends inside 16 bytes writes the rest of them too.)
  p.tma_store = r.split == 1 && a->m > 0 && rows_16b(a->d, a->ldd, e) && (a->n * e) % 16 == 0 ? 1 : 0;
  p.stg_bufs = p.tma_store ? 2 : 0;
  p.c_staged = p.tma_store && a->c && rows_16b(a->c, a->ldc, e) ? 1 : 0;
  p.c_bufs = kCBufs;
  if (p.c_staged) p.stg_bufs = p.c_bufs;
  // A second epilogue group where the main loop is too short to hide one, and where it shares
  // the accumulator's columns with the next tile, which then waits for one chunk of each group.
  p.groups = r.cg == 2 && (r.bn == 256 || p.num_kb < (p.c ? 40 : 20)) ? 2 : 1;
  const int kb_cta = (p.num_kb + r.split - 1) / r.split;
  const int64_t tok_bytes = fused ? (int64_t)(kb_cta + 1) * kTokAtom : 0;
  const int64_t tok_tiles = fused ? ((int64_t)kb_cta * sf * kTokTile + 384 + 511) / 512 * 512 : 0;
  const int64_t fixed = 1024 + kBarrierBytes + (int64_t)p.groups * p.stg_bufs * p.stg_bytes + p.groups * 4 * r.bn * 4 + tok_bytes + tok_tiles + kStaticSmem;
  r.max_stages = (int)((kSmemLimit - fixed) / p.stage_bytes);
  if (r.max_stages > kMaxStages4) r.max_stages = kMaxStages4;
  // (No tile but that of 256 tokens has more stages than slots as it is.)
  if (r.bn != 256 && r.max_stages > scale_slots(r.bn, a->block)) r.max_stages = scale_slots(r.bn, a->block);
  r.stages = r.max_stages;
  if (r.split > 1) {
    if (r.stages > kb_cta) r.stages = kb_cta;
    while ((int64_t)r.stages * p.stage_bytes < (int64_t)r.bn * kChannels * 4) ++r.stages;   // the partial tile lies over the ring
  }
  p.stages = r.stages;
  p.bars_offset = (uint32_t)r.stages * p.stage_bytes;
  p.tok_offset = p.bars_offset + kBarrierBytes;
  p.tok_tiles = p.tok_offset + (uint32_t)tok_bytes;
  p.stg_offset = p.tok_tiles + (uint32_t)tok_tiles;
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

using KernelFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Fp4Params);

template <int BLOCK, typename T>
KernelFn pick(int cg, int bn, bool fused) {
  if (fused) return fp4_gemm_kernel<1, kFusedBN, BLOCK, T, true>;
  if (cg == 1) {
    switch (bn) {
      case 16: return fp4_gemm_kernel<1, 16, BLOCK, T, false>;
      case 32: return fp4_gemm_kernel<1, 32, BLOCK, T, false>;
      case 64: return fp4_gemm_kernel<1, 64, BLOCK, T, false>;
      default: return fp4_gemm_kernel<1, 128, BLOCK, T, false>;
    }
  }
  return bn == 128 ? fp4_gemm_kernel<2, 128, BLOCK, T, false> : fp4_gemm_kernel<2, 256, BLOCK, T, false>;
}
KernelFn pick(const Fp4GemmArgs& a, const Resolved& r, bool fused) {
  if (a.block == 16)
    return a.d_type == GEMM_TYPE_BF16 ? pick<16, __nv_bfloat16>(r.cg, r.bn, fused) : pick<16, __half>(r.cg, r.bn, fused);
  return a.d_type == GEMM_TYPE_BF16 ? pick<32, __nv_bfloat16>(r.cg, r.bn, fused) : pick<32, __half>(r.cg, r.bn, fused);
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

// Scale tiles as words: 128 to a tile, tiles along a row, row blocks.
bool encode_tiles(CUtensorMap* m, const void* ptr, int64_t tiles, int64_t row_blocks, int box_tiles, int box_blocks) {
  cuuint64_t dims[3] = {128, (cuuint64_t)tiles, (cuuint64_t)row_blocks};
  cuuint64_t strides[2] = {512, (cuuint64_t)tiles * 512};
  cuuint32_t box[3] = {128, (cuuint32_t)box_tiles, (cuuint32_t)box_blocks};
  cuuint32_t estr[3] = {1, 1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Tokens {        // floating tokens of the fused form
  const void* x;
  int64_t ldx;
};

// A product that is ready to be launched: nothing can refuse it any more.
struct Prepared {
  Resolved r;
  CUtensorMap tw, tt, td, tc, tws, tts;
  KernelFn fn;
  int threads;
};

// The device of D is current.
int prepare_product(const Fp4GemmArgs& a, const Tokens* tokens, int dev, Prepared& q) {
  Resolved& r = q.r;
  const int rc = resolve(&a, tokens != nullptr, r);
  if (rc != GEMM_OK) return rc;
  if (!get_encode()) return GEMM_ERR_LAUNCH;
  memset(&q.tt, 0, sizeof(q.tt));
  memset(&q.td, 0, sizeof(q.td));
  memset(&q.tc, 0, sizeof(q.tc));
  memset(&q.tws, 0, sizeof(q.tws));
  memset(&q.tts, 0, sizeof(q.tts));
  const uint64_t row_bytes = (uint64_t)(a.k + 1) / 2;
  if (!encode_2d(&q.tw, a.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, row_bytes, (uint64_t)a.n, (uint64_t)a.ldb, kAtom, kChannels, 128))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (tokens) {
    r.p.x = tokens->x;
    r.p.ldx = tokens->ldx;
  } else if (!encode_2d(&q.tt, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, row_bytes, (uint64_t)a.m, (uint64_t)a.lda, kAtom,
                        (uint32_t)(r.bn / r.cg), 128)) {
    return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  if (r.cg == 2) {
    const int sf = tiles_per_atom(a.block);
    if (!encode_tiles(&q.tws, a.b_scales, r.p.tiles, (a.n + 127) / 128, sf, 1) ||
        !encode_tiles(&q.tts, a.a_scales, r.p.tiles, (a.m + 127) / 128, sf, (r.bn + 127) / 128))
      return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  if (r.p.tma_store) {
    const CUtensorMapDataType t = a.d_type == GEMM_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint32_t tokens_box = (uint32_t)(r.bn < 32 ? r.bn : 32);
    if (!encode_2d(&q.td, a.d, t, (uint64_t)a.n, (uint64_t)a.m, (uint64_t)(a.ldd * 2), kChannels, tokens_box, 0))
      return GEMM_ERR_CANNOT_IMPLEMENT;
    if (r.p.c_staged && !encode_2d(&q.tc, a.c, t, (uint64_t)a.n, (uint64_t)a.m, (uint64_t)(a.ldc * 2), kChannels, tokens_box, 0))
      return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  q.fn = pick(a, r, tokens != nullptr);
  q.threads = tokens ? threads_for(1, true) : 64 + 128 * r.p.groups;
  return ensure_smem_attr(q.fn, dev, tokens ? kSmemLimit - kStaticSmem : kSmemLimit) ? GEMM_OK : GEMM_ERR_LAUNCH;
}

int launch_prepared(const Prepared& q, cudaStream_t st) {
  const Resolved& r = q.r;
  if (launch_overlapped(q.fn, dim3((unsigned)r.grid), dim3((unsigned)q.threads), (size_t)r.smem_bytes,
                        r.split > 1 ? r.split : r.cg, st, q.tw, q.tt, q.td, q.tc, q.tws, q.tts, r.p) != cudaSuccess) {
    cudaGetLastError();
    return GEMM_ERR_LAUNCH;
  }
  return GEMM_OK;
}

// Few tokens, no knob set and X of D's type: one launch.  One token x 8192 x 8192 takes 10.6 us a call that way and 13.7 in two
// launches, 8 tokens x 2048 x 8192 6.5 and 8.3.  (From a graph, where a launch costs less than every CTA's own
// quantisation, 6.2 and 5.8 for the latter: a knob makes two launches of it.)  A D that lies over the tokens (the layer's result
// replaces them) needs two launches, the tokens being quantised before the first store.
bool use_fused(const Fp4GemmArgs& a, const void* x, int32_t x_type, int64_t ldx) {
  if (a.m > kFusedTokens || a.m < 1 || a.n < 1 || a.k < 1 || a.k > kFusedElems) return false;
  if (a.m * ((a.k + kAtomK - 1) / kAtomK * kAtomK) > kFusedElems || x_type != a.d_type || a.tile_n || a.cta_group || a.split_k || a.flags)
    return false;
  const int64_t e = type_bytes(x_type);
  return !rows_meet(x, ldx * e, a.k * e, a.d, a.ldd * e, a.n * e, a.m);
}

}  // namespace

extern "C" int gemm_sm100a_fp4_query(const Fp4GemmArgs* args, GemmInfo* info) {
  Resolved r;
  const int rc = resolve(args, false, r);
  if (info) {
    memset(info, 0, sizeof(*info));
    info->struct_size = sizeof(GemmInfo);
    info->tile_m = kChannels * r.cg; info->tile_n = r.bn; info->tile_k = kAtomK; info->stages = r.stages;
    info->cta_group = r.cg; info->cluster_m = r.split > 1 ? r.split : r.cg; info->max_stages = r.max_stages;
    info->smem_bytes_per_stage = r.p.stage_bytes; info->smem_bytes = r.smem_bytes;
    info->tmem_columns = kTmemCols; info->grid_ctas = r.grid; info->num_tiles = r.p.num_units;
    info->num_sms = r.num_sms; info->can_implement = rc == GEMM_OK;
    memcpy(info->reason, r.reason, sizeof(info->reason));
    info->epilogue_staging_buffers = r.p.stg_bufs;
  }
  return rc;
}

extern "C" int gemm_sm100a_fp4_launch(const Fp4GemmArgs* args, void* stream) {
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

extern "C" int gemm_sm100a_fp4_linear_workspace(const Fp4GemmArgs* args, const void* x, int32_t x_type, int64_t ldx) {
  return args && args->struct_size == sizeof(Fp4GemmArgs) && use_fused(*args, x, x_type, ldx) ? 0 : 1;
}

extern "C" int gemm_sm100a_fp4_linear(const Fp4GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream) {
  Resolved r;
  memset(&r, 0, sizeof(r));
  const bool few = gemm_sm100a_fp4_linear_workspace(args, x, x_type, ldx) == 0;
  const int rc = check(args, !few, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  if (!type_ok(x_type)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!x || (!few && !args->a_row_scale)) return GEMM_ERR_BAD_ARGS;
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
    Fp4QuantArgs q;
    memset(&q, 0, sizeof(q));
    q.struct_size = sizeof(q);
    q.x_type = x_type; q.rows = args->m; q.cols = args->k; q.x = x; q.ldx = ldx; q.block = args->block;
    q.values = const_cast<void*>(args->a); q.ldv = args->lda;
    q.scales = const_cast<void*>(args->a_scales); q.row_scale = const_cast<float*>(args->a_row_scale);
    const int rq = gemm_sm100a_quantize_fp4(&q, stream);
    if (rq != GEMM_OK) return rq;
  }
  return launch_prepared(p, st);
}
