// residual_norm.cu -- the residual stream around a block: the norm after it, its gate and scale, the stream's
// update and the norm before the next block, and their gradients.  Bound by the bytes of the rows: four
// matrices forward (three and a quarter where the result becomes a 4-bit operand), six backward.
//
//   z = y r(y) wp,  x' = x + (gate scale) z,  h = x' r(x') w,  r(v) = 1 / sqrt(mean(v^2) + eps)
//
// Backward, with n columns, dn = dh w, k = gate scale, P = k wp y, r = r(x'), q = r(y):
//   g  = dx' + r dn - x' r^3 (sum dn x') / n
//   dy = q (k wp g - y q^2 (sum P g) / n)
//   sum P g = sum P dx' + r sum P dn - r^3 (sum dn x') / n sum P x'
// so that all row sums (with those of x'^2 and y^2) come from one pass and one exchange, and no statistics are
// kept from the forward call.  The sums over rows (dw, dwp, dgate) stay with the threads of a CTA, which walks down the
// matrix; the CTAs' parts go through a workspace to a second kernel that adds them in order.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "fp4_common.cuh"
#include "gemm_sm100a.h"
#include "row_stream.cuh"
#include "sm100_ptx.cuh"

using namespace int8op;
using rowvec::kUnit;
using rowvec::Unit;
using namespace rowstream;

namespace {

constexpr int kMaxCols = 16384;
constexpr int kManyThreads = 768;          // of a forward block of many rows
template <typename T>
constexpr int many_threads() { return sizeof(T) == 2 ? kManyThreads : kMaxThreads; }

// ----------------------------------------------------------------- statistics
template <typename T>
__device__ __forceinline__ F2 pair(const Unit<T>& u, int j) { return F2(u.get(2 * j), u.get(2 * j + 1)); }
__device__ __forceinline__ float both(F2 v) {
  float a, b;
  v.get(a, b);
  return a + b;
}
__device__ __forceinline__ F2 f2(float v) { return F2(v, v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ float squares(const Unit<T>& u) {
  F2 s = f2(0.f);
#pragma unroll
  for (int j = 0; j < kUnit / 2; ++j) s = fma2(pair(u, j), pair(u, j), s);
  return both(s);
}
template <typename T>
__device__ __forceinline__ double squares_wide(const Unit<T>& u) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kUnit; ++j) s = fma((double)u.get(j), (double)u.get(j), s);
  return s;
}
// Where the fp32 part of a sum of squares may have left its range (or come near its end), 64 bits do it again.
__device__ __forceinline__ bool out_of_range(float s) { return !(s > 1e-30f && s < 1e38f); }

// 1 / sqrt(v), rounded to fp32 from an error of 2^-43 or so: one Newton step whose 1 - v r^2 has v and r^2 in two fp32
// words each.
__device__ __forceinline__ float inverse_root(double v) {
  if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
  const float hi = (float)v, lo = (float)(v - (double)hi);
  const float r = rsqrtf(hi), p = r * r, p_lo = fmaf(r, r, -p);
  const float t = fmaf(-hi, p, 1.f) - fmaf(hi, p_lo, lo * p);
  return fmaf(0.5f * r, t, r);
}

// The sum over the group's threads; all of them call, with `part` alternating between calls.
__device__ __forceinline__ float group_sum(float v, float* part) {
  v = warp_sum(v);
  const int warps = (int)blockDim.x >> 5, lane = (int)(threadIdx.x & 31u);
  if (warps == 1) return v;
  float* const mine = part + threadIdx.y * warps;
  if (lane == 0) mine[threadIdx.x >> 5] = v;
  group_sync();
  return warp_sum(lane < warps ? mine[lane] : 0.f);
}
// The sum over the group's warps of a value that the lanes of each warp hold, in 64 bits.
__device__ __forceinline__ double across_warps(double v, double* part) {
  const int warps = (int)blockDim.x >> 5;
  if (warps == 1) return v;
  double* const mine = part + threadIdx.y * warps;
  if ((threadIdx.x & 31u) == 0) mine[threadIdx.x >> 5] = v;
  group_sync();
  double s[2] = {0.0, 0.0};
#pragma unroll 4
  for (int i = 0; i < warps; ++i) s[i & 1] += mine[i];
  return s[0] + s[1];
}

struct NormParams {
  const uint8_t* x; int64_t ldx;       // strides in bytes
  const uint8_t* y; int64_t ldy;
  uint8_t* xo; int64_t ldo;
  uint8_t* h; int64_t ldh;
  const void* w;
  const void* wp;
  const uint8_t* gate; int64_t ldg;
  int64_t rows;
  int32_t cols;
  float scale;
  double eps, inv_n;
  uint8_t* values; int64_t ldv;
  uint8_t* scales;
  float* row_scale;
  int64_t tiles;
  int32_t stages;              // rows ahead
  uint32_t place;              // bytes of a stretch in shared memory
  int32_t gate_ahead;          // a gate matrix is copied ahead too
  int32_t param32;             // the vectors are fp32 (else of T)
  int32_t vectors_at;          // many rows: byte of the vectors in shared memory
  int32_t block;               // of the 4-bit form
};

// A vector's elements at a thread's unit as fp32 pairs; ones where there is no vector.
template <typename T>
__device__ __forceinline__ void load_params(const void* v, int param32, int e, int n, F2 (&o)[kUnit / 2]) {
  if (!v) {
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = f2(1.f);
  } else if (sizeof(T) == 4 || param32) {
    const Unit<float> u = rowvec::load_unit<float, rowvec::kKeep>(static_cast<const float*>(v) + e, n);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = pair(u, j);
  } else {
    const Unit<T> u = rowvec::load_unit<T, rowvec::kKeep>(static_cast<const T*>(v) + e, n);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) o[j] = pair(u, j);
  }
}

// Vectors that all groups of a block read, in shared memory: four elements of a unit to a slot, the slots of one kind side by
// side for all units (no bank conflicts).
struct SharedVectors {
  uint32_t base, per_chunk;      // bytes from a unit's slot to that of its next four elements
  __device__ __forceinline__ uint32_t at(int which, int unit) const { return base + (uint32_t)(which * 4) * per_chunk + (uint32_t)unit * 16u; }
  __device__ __forceinline__ void put(int which, int unit, const F2 (&v)[kUnit / 2]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float f[4];
      v[2 * c].get(f[0], f[1]);
      v[2 * c + 1].get(f[2], f[3]);
      sm100::st_shared_v4(at(which, unit) + (uint32_t)c * per_chunk, __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
  }
  // Pairs 2 c and 2 c + 1 of a unit.
  __device__ __forceinline__ void get(int which, int unit, int c, F2& a, F2& b) const {
    const uint4 u = sm100::ld_shared_v4(at(which, unit) + (uint32_t)c * per_chunk);
    a = F2(__uint_as_float(u.x), __uint_as_float(u.y));
    b = F2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  __device__ __forceinline__ void get(int which, int unit, F2 (&v)[kUnit / 2]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) get(which, unit, c, v[2 * c], v[2 * c + 1]);
  }
};

// NU units to a thread, blockDim.x units apart.
//  Few rows (NU 1): the vectors stay in registers.
//  Many rows (NU 2, which halves what the statistics cost per element): the vectors lie in shared memory as w and wp gate scale,
//    in fp32, where all groups of the block read them, and up to four groups of 8192-element rows hide one another's
//    barriers.  Rows that leave no room for them read them from the caches each time.
// KIND 0: no y; 1: y; 2: y and a gate matrix.  (What can be absent from call to call is decided here where
// the compiler would otherwise make a copy of the loop for each case, with the registers of all.)
template <typename T, bool FOUR, int NU, bool FULL, int KIND>
__global__ void __launch_bounds__(NU == 2 ? many_threads<T>() : kMaxThreads, 1) residual_norm_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ double part[2][kManyThreads / 32];
  __shared__ float part32[2][kManyThreads / 32];
  __shared__ uint32_t warp_max[kManyThreads / 32];
  constexpr int E = (int)sizeof(T);
  constexpr bool KEEP = NU == 1, SHARED = NU == 2 && E == 2, BLOCK = KIND > 0, MATRIX = KIND == 2;
  const int tx = threadIdx.x, TX = blockDim.x;
  // Places of this warp: stage by stage, then unit by unit, then matrix by matrix.
  const uint32_t per_unit = p.place, per_stage = (uint32_t)(((BLOCK ? 2 : 1) + (MATRIX ? p.gate_ahead : 0)) * NU) * per_unit;
  const uint32_t mine = sm100::smem_u32(slots) + (uint32_t)((int)threadIdx.y * (TX >> 5) + (tx >> 5)) * (uint32_t)p.stages * per_stage;
  const int lane_e = (tx & 31) * kUnit;       // elements from a warp's first unit to this lane's
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, step = (int64_t)gridDim.x * blockDim.y;
  int e[NU], n[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    e[i] = (i * TX + tx) * kUnit;
    n[i] = p.cols - e[i];
  }
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  auto issue = [&](int64_t row, uint32_t slot) {
    if (row < p.rows) {
      const uint8_t* const rx = row_of(p.x, row, p.ldx);
      const uint8_t* const ry = row_of(p.y, row, p.ldy);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        issue_stretch<T, FULL>(slot, rx + (e[i] - lane_e) * E, n[i] + lane_e);
        slot += per_unit;
        if (BLOCK) {
          issue_stretch<T, FULL>(slot, ry + (e[i] - lane_e) * E, n[i] + lane_e);
          slot += per_unit;
        }
        if (MATRIX && p.gate_ahead) {
          issue_stretch<T, FULL>(slot, row_of(p.gate, row, p.ldg) + (e[i] - lane_e) * E, n[i] + lane_e);
          slot += per_unit;
        }
      }
    }
    commit_copies();
  };
  for (int s = 0; s < p.stages; ++s) issue(first + s * step, mine + (uint32_t)s * per_stage);

  F2 vw[kUnit / 2], vk[kUnit / 2];
  auto load_w = [&](int i) { load_params<T>(p.w, p.param32, e[i], n[i], vw); };
  auto load_k = [&](int i) {
    F2 g[kUnit / 2];
    load_params<T>(p.wp, p.param32, e[i], n[i], vk);
    load_params<T>(MATRIX ? nullptr : p.gate, p.param32, e[i], n[i], g);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) vk[j] = mul2(vk[j], mul2(g[j], f2(p.scale)));
  };
  const SharedVectors vectors = {sm100::smem_u32(slots) + (uint32_t)p.vectors_at, (uint32_t)(NU * TX) * 16u};
  if constexpr (KEEP) {
    load_w(0);
    if (BLOCK) load_k(0);
  } else if (SHARED) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (((int)threadIdx.y - i) % (int)blockDim.y == 0 || blockDim.y == 1) {
        load_w(i);
        vectors.put(0, i * TX + tx, vw);
        if (BLOCK) {
          load_k(i);
          vectors.put(1, i * TX + tx, vk);
        }
      }
    }
    __syncthreads();
  }

  int flip = 0;       // a call's buffer is written again by the second call after it, with a barrier between
  auto inverse_rms = [&](const Unit<T> (&v)[NU]) {
    double* const at = part[flip ^= 1];
    double s = 0.0;
    if constexpr (E == 4) {
#pragma unroll
      for (int i = 0; i < NU; ++i) s += squares_wide<T>(v[i]);
      s = across_warps(warp_sum(s), at);
    } else {
      // In fp32, pairwise from a few elements up: 64 bits cost the kernel of 16-bit elements twice its instructions for a last
      // bit of r that their results do not show.
      float f = 0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i) f += squares<T>(v[i]);
      f = group_sum(f, part32[flip]);
      if (!out_of_range(f)) {
        const float m = fmaf(f, (float)p.inv_n, (float)p.eps), r = rsqrtf(m);
        return fmaf(0.5f * r, fmaf(-m * r, r, 1.f), r);
      } else {
        group_sync();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < NU; ++i) s += squares_wide<T>(v[i]);
        s = across_warps(warp_sum(s), at);
      }
    }
    return inverse_root(fma(s, p.inv_n, p.eps));
  };

  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const uint32_t at = mine + (uint32_t)stage * per_stage;
    const uint8_t* const rx = p.x + row * p.ldx;
    const uint8_t* const ry = p.y + row * p.ldy;
    const uint8_t* const rg = p.gate + row * p.ldg;
    auto low = [](const uint8_t* q) { return (uint32_t)reinterpret_cast<uintptr_t>(q) & 15u; };      // (units are multiples of 16 bytes)
    wait_copies(p.stages - 1);
    __syncwarp();
    Unit<T> x[NU], y[NU], gate[NU];
    {
      uint32_t slot = at;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        x[i] = take_unit<T, FULL>(slot, low(rx), n[i]);
        slot += per_unit;
        if (BLOCK) {
          y[i] = take_unit<T, FULL>(slot, low(ry), n[i]);
          slot += per_unit;
        }
        if (MATRIX && p.gate_ahead) {
          gate[i] = take_unit<T, FULL>(slot, low(rg), n[i]);
          slot += per_unit;
        } else if (MATRIX) {
          gate[i] = rowvec::load_unit<T>(reinterpret_cast<const T*>(rg) + e[i], n[i]);
        }
      }
    }
    __syncwarp();
    issue(row + p.stages * step, at);
    if (++stage == p.stages) stage = 0;
    if constexpr (BLOCK) {
      const F2 q = f2(p.wp ? inverse_rms(y) : 1.f);
#pragma unroll
      for (int i = 0; i < NU; ++i) forget(y[i]);
      uint8_t* const out = row_of(p.xo, row, p.ldo);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (!KEEP && !SHARED) load_k(i);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          F2 k[2] = {vk[2 * c], vk[2 * c + 1]};
          if (SHARED) vectors.get(1, i * TX + tx, c, k[0], k[1]);
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            const int j = 2 * c + l;
            if (MATRIX) k[l] = mul2(k[l], pair(gate[i], j));
            float a, b;
            fma2(mul2(pair(y[i], j), q), k[l], pair(x[i], j)).get(a, b);
            x[i].set2(2 * j, a, b);
          }
        }
        put_unit<T, FULL>(out + e[i] * E, x[i], n[i]);
      }
    }
    const F2 r = f2(inverse_rms(x));
#pragma unroll
    for (int i = 0; i < NU; ++i) forget(x[i]);
    // h of a unit, in fp32.
    auto norm = [&](int i, float (&h)[kUnit]) {
      if (!KEEP && !SHARED) load_w(i);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        F2 w[2] = {vw[2 * c], vw[2 * c + 1]};
        if (SHARED) vectors.get(0, i * TX + tx, c, w[0], w[1]);
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          const int j = 2 * c + l;
          mul2(mul2(pair(x[i], j), r), w[l]).get(h[2 * j], h[2 * j + 1]);
        }
      }
    };
    if constexpr (!FOUR) {
      uint8_t* const out = row_of(p.h, row, p.ldh);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        float h[kUnit];
        norm(i, h);
        Unit<T> o;
#pragma unroll
        for (int j = 0; j < kUnit; j += 2) o.set2(j, h[j], h[j + 1]);
        put_unit<T, FULL>(out + e[i] * E, o, n[i]);
      }
    } else {
      float h[NU][kUnit], tops[NU];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        norm(i, h[i]);
        if (n[i] < kUnit) {
          // Zeros beyond the row (an infinite r has made NaN of them).
#pragma unroll
          for (int j = 0; j < kUnit; ++j)
            if (j >= n[i]) h[i][j] = 0.f;
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) m = max(m, __float_as_uint(h[i][j]) & 0x7FFFFFFFu);
        tops[i] = __uint_as_float(m);
        top = max(top, m);
      }
      top = __reduce_max_sync(0xFFFFFFFFu, top);
      if (TX > 32) {
        // (The barrier of the next row's statistics lies between this row's reads and that row's writes.)
        uint32_t* const group = warp_max + (int)threadIdx.y * (TX >> 5);
        if ((tx & 31) == 0) group[tx >> 5] = top;
        group_sync();
        top = __reduce_max_sync(0xFFFFFFFFu, (tx & 31) < (TX >> 5) ? group[tx & 31] : 0u);
      }
      const fp4op::RowScale s = fp4op::row_scale(top);
      if (tx == 0) p.row_scale[row] = s.scale;
      const bool far = s.far();
      const float up = far ? 1.f : s.up, unit_g = far ? 1.f : s.scale;
      const int units = (int)p.tiles * 4 * (p.block / 16);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int unit = i * TX + tx;
        if ((unit & ~31) >= units) break;      // whole warps
        if (far) fp4op::bring_near(h[i], tops[i], s);
        uint32_t q[2];
        if (p.block == 16) fp4op::store_scale_codes<16>(p.scales, row, p.tiles, unit, fp4op::quantize_unit<16>(h[i], tops[i], up, unit_g, q), unit < units);
        else fp4op::store_scale_codes<32>(p.scales, row, p.tiles, unit, fp4op::quantize_unit<32>(h[i], tops[i], up, unit_g, q), unit < units);
        if (n[i] > 0) fp4op::store_codes(p.values + row * p.ldv + unit * 8, q, n[i]);
      }
    }
  }
}

bool rows_wide(const NormParams& p) { return all_wide({{p.x, p.ldx}, {p.y, p.ldy}, {p.ldg ? p.gate : nullptr, p.ldg}}); }

template <typename T, bool FOUR, int NU, bool FULL, int KIND>
cudaError_t launch_forward(const NormParams& p0, cudaStream_t st) {
  NormParams p = p0;
  constexpr bool SHARED = NU == 2 && sizeof(T) == 2;
  const int units = FOUR ? (int)p.tiles * 4 * (p.block / 16) : (p.cols + kUnit - 1) / kUnit;
  p.place = place_bytes((int)sizeof(T), FULL || rows_wide(p));
  const int two = (KIND ? 2 : 1) * NU * (int)p.place, three = two + (KIND == 2 ? NU * (int)p.place : 0);
  const int tx = ((units + NU - 1) / NU + 31) / 32 * 32, vectors = SHARED ? tx * NU * kUnit * 4 * (KIND ? 2 : 1) : 0;
  // A gate matrix is not copied ahead where there is no room for it (rows of more than some 14000 elements).
  p.gate_ahead = KIND == 2 && vectors + three * (tx / 32) <= kSmemLimit;
  const Shape s = shape_of(p.rows, units, NU, p.gate_ahead ? three : two, NU == 2 ? many_threads<T>() : kMaxThreads, vectors);
  if (s.stages < 1) return cudaErrorInvalidValue;
  p.stages = s.stages;
  p.vectors_at = (int32_t)s.smem;
  const auto fn = residual_norm_kernel<T, FOUR, NU, FULL, KIND>;
  // (Always the same limit: calls of other sizes may be between this line and the launch.)
  const cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (err != cudaSuccess) return err;
  return launch_overlapped(fn, dim3((unsigned)s.blocks), dim3((unsigned)s.tx, (unsigned)s.ty), s.smem + vectors, 1, st, p);
}
template <typename T, bool FOUR, int KIND>
cudaError_t launch_forward(const NormParams& p, cudaStream_t st) {
  if (p.cols <= kMaxThreads * kUnit && p.rows <= 148) return launch_forward<T, FOUR, 1, false, KIND>(p, st);
  const bool wide = rows_wide(p) && all_wide({{p.xo, p.ldo}, {p.h, p.ldh}}) && all_full((p.cols + kUnit - 1) / kUnit, p.cols, 2);
  return wide ? launch_forward<T, FOUR, 2, true, KIND>(p, st) : launch_forward<T, FOUR, 2, false, KIND>(p, st);
}
template <typename T>
cudaError_t launch_forward(const NormParams& p, cudaStream_t st) {
  const int kind = !p.y ? 0 : p.ldg ? 2 : 1;
  if (p.block) return kind == 0 ? launch_forward<T, true, 0>(p, st) : kind == 1 ? launch_forward<T, true, 1>(p, st) : launch_forward<T, true, 2>(p, st);
  return kind == 0 ? launch_forward<T, false, 0>(p, st) : kind == 1 ? launch_forward<T, false, 1>(p, st) : launch_forward<T, false, 2>(p, st);
}

// ----------------------------------------------------------------- backward
struct BackParams {
  const uint8_t* in[5]; int64_t ld[5];   // x_out, dh, dx_out, y, gate (strides in bytes; NULL where absent, the gate where it is no matrix)
  const void* w;
  const void* wp;
  const void* gate;                      // as a vector
  uint8_t* dx; int64_t lddx;
  uint8_t* dy; int64_t lddy;
  uint8_t* dgate; int64_t lddg;          // matrix; NULL where it is a vector
  float* parts;                          // [block][2][cols]
  int64_t rows;
  int32_t cols;
  float scale;
  double eps, inv_n;
  int32_t stages;
  uint32_t place;
  int32_t param32;
  int32_t vectors_at;
};

// Row sums: 0 x^2, 1 y^2, 2 dn x, 3 P dx', 4 P dn, 5 P x.
struct BackSums {
  float part[kMaxThreads / 32][8];
  double wide[2][kMaxThreads / 32];
  float4 row[8];                 // r, q and the two coefficients, one row to a group
};

// Sums over the warp of eight values per lane: lane l ends with the one of index l / 4.
__device__ __forceinline__ float warp_sums(float (&v)[8]) {
  const int lane = (int)(threadIdx.x & 31u);
#pragma unroll
  for (int half = 4; half > 0; half /= 2) {
    const bool upper = lane & (4 * half);
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, 4 * half);
    }
  }
  float s = v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 2);
  return s + __shfl_xor_sync(0xFFFFFFFFu, s, 1);
}

// As in the forward kernel: NU units to a thread, the vectors in registers (NU 1) or shared memory (NU 2), the coming row on its
// way while other groups are at work.  A row stays in shared memory for both of its passes.
//  HELD (rows of more than 8192 elements): two units, rows read twice from global memory (the second time from the
// caches) and the column sums in shared memory.
//  The column sums are two: of dh x r, and of g y q (times a gate matrix' k): dpost and a vector's dgate are the second
// times what their columns share.
//  KIND 0: no y; 1: y; 2: y and its norm; 3, 4: 1, 2 with a gate matrix.
template <typename T, int NU, bool HELD, bool FULL, int KIND>
__global__ void __launch_bounds__(kMaxThreads, 1) residual_norm_backward_kernel(const __grid_constant__ BackParams p) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ BackSums sums;
  float* const held = reinterpret_cast<float*>(slots);       // [2][cols rounded up to units]
  constexpr int E = (int)sizeof(T);
  constexpr bool BLOCK = KIND > 0, POST = KIND == 2 || KIND == 4, MATRIX = KIND > 2, SHARED = NU == 2 && !HELD;
  enum { X, DH, DX, Y, G };
  const int tx = threadIdx.x, TX = blockDim.x;
  const int width = (p.cols + kUnit - 1) / kUnit * kUnit;
  const uint32_t per_stage = (uint32_t)((BLOCK ? 4 : 3) + (MATRIX ? 1 : 0)) * NU * p.place;
  const uint32_t mine = sm100::smem_u32(slots) + (uint32_t)((int)threadIdx.y * (TX >> 5) + (tx >> 5)) * (uint32_t)p.stages * per_stage;
  auto unit_at = [&](int i) { return (i * TX + tx) * kUnit; };
  if constexpr (HELD) {
    for (int i = tx; i < 2 * width; i += TX) held[i] = 0.f;
    __syncthreads();
  }
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, step = (int64_t)gridDim.x * blockDim.y;
  auto issue = [&](int64_t row, uint32_t slot) {
    if (row < p.rows) {
#pragma unroll
      for (int m = 0; m < 5; ++m) {
        if ((m == Y && !BLOCK) || (m == G && !MATRIX)) continue;
        const uint8_t* const r = row_of(p.in[m], row, p.ld[m]);
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          const int e = unit_at(i) - (tx & 31) * kUnit;
          if (m != DX || each_row(p.in[DX])) issue_stretch<T, FULL>(slot, r + e * E, p.cols - e);
          slot += p.place;
        }
      }
    }
    commit_copies();
  };
  if constexpr (!HELD)
    for (int s = 0; s < p.stages; ++s) issue(first + s * step, mine + (uint32_t)s * per_stage);

  F2 vw[kUnit / 2], vk[kUnit / 2];       // w, and k wp (wp scale with a gate matrix)
  auto load_vectors = [&](int i) {
    const int e = unit_at(i);
    F2 k[kUnit / 2];
    load_params<T>(p.w, p.param32, e, p.cols - e, vw);
    load_params<T>(p.wp, p.param32, e, p.cols - e, vk);
    load_params<T>(p.gate, p.param32, e, p.cols - e, k);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) vk[j] = mul2(vk[j], mul2(k[j], f2(p.scale)));
  };
  const SharedVectors vectors = {sm100::smem_u32(slots) + (uint32_t)p.vectors_at, (uint32_t)(NU * TX) * 16u};
  if constexpr (SHARED) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (((int)threadIdx.y - i) % (int)blockDim.y == 0 || blockDim.y == 1) {
        load_vectors(i);
        vectors.put(0, i * TX + tx, vw);
        vectors.put(1, i * TX + tx, vk);
      }
    }
    __syncthreads();
  } else if constexpr (!HELD) {
    load_vectors(0);
  }
  F2 cw[NU][kUnit / 2], cs[NU][kUnit / 2];
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) cw[i][j] = cs[i][j] = f2(0.f);
  const float inv_n = (float)p.inv_n;
  const int warps = TX >> 5, first_warp = (int)threadIdx.y * warps, lane = tx & 31;

  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const uint32_t at = mine + (uint32_t)stage * per_stage;
    if constexpr (!HELD) {
      wait_copies(p.stages - 1);
      __syncwarp();
    }
    auto get = [&](int m, int i) {
      const int e = unit_at(i), n = p.cols - e;
      Unit<T> u;
      if (m == DX && each_row(!p.in[DX])) u.clear();
      else if constexpr (HELD) u = rowvec::load_unit<T, rowvec::kKeep>(reinterpret_cast<const T*>(row_of(p.in[m], row, p.ld[m])) + e, n);
      else u = take_unit<T, FULL>(at + (uint32_t)(m * NU + i) * p.place, FULL ? 0u : (uint32_t)reinterpret_cast<uintptr_t>(p.in[m] + row * p.ld[m]) & 15u, n);
      return u;
    };
    // ---- row sums
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if constexpr (HELD) load_vectors(i);
      if constexpr (SHARED) vectors.get(0, i * TX + tx, vw);
      const Unit<T> x = get(X, i), dh = get(DH, i);
      F2 s0 = f2(0.f), s2 = f2(0.f);
      if constexpr (!POST) {
#pragma unroll
        for (int j = 0; j < kUnit / 2; ++j) {
          const F2 xv = pair(x, j);
          s0 = fma2(xv, xv, s0);
          s2 = fma2(mul2(pair(dh, j), vw[j]), xv, s2);
        }
      } else {
        const Unit<T> y = get(Y, i), d = get(DX, i);
        Unit<T> g;
        if constexpr (MATRIX) g = get(G, i);
        if constexpr (SHARED) vectors.get(1, i * TX + tx, vk);
        F2 s1 = f2(0.f), s3 = f2(0.f), s4 = f2(0.f), s5 = f2(0.f);
#pragma unroll
        for (int j = 0; j < kUnit / 2; ++j) {
          const F2 xv = pair(x, j), yv = pair(y, j), dn = mul2(pair(dh, j), vw[j]);
          s0 = fma2(xv, xv, s0);
          s1 = fma2(yv, yv, s1);
          s2 = fma2(dn, xv, s2);
          F2 f = mul2(vk[j], yv);
          if constexpr (MATRIX) f = mul2(f, pair(g, j));
          s3 = fma2(f, pair(d, j), s3);
          s4 = fma2(f, dn, s4);
          s5 = fma2(f, xv, s5);
        }
        v[1] += both(s1);
        v[3] += both(s3);
        v[4] += both(s4);
        v[5] += both(s5);
      }
      v[0] += both(s0);
      v[2] += both(s2);
    }
    const float s = warp_sums(v);
    if ((lane & 3) == 0) sums.part[first_warp + (tx >> 5)][lane >> 2] = s;
    group_sync();
    // The group's first warp adds the warps' sums: lane l the values 4 (l & 1) .. + 3 of warp l / 2.
    if (tx < 32) {
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if ((lane >> 1) < warps) t = *reinterpret_cast<const float4*>(&sums.part[first_warp + (lane >> 1)][4 * (lane & 1)]);
#pragma unroll
      for (int o = 2; o < 32; o *= 2) {
        t.x += __shfl_xor_sync(0xFFFFFFFFu, t.x, o);
        t.y += __shfl_xor_sync(0xFFFFFFFFu, t.y, o);
        t.z += __shfl_xor_sync(0xFFFFFFFFu, t.z, o);
        t.w += __shfl_xor_sync(0xFFFFFFFFu, t.w, o);
      }
      const float b2 = __shfl_sync(0xFFFFFFFFu, t.x, 1), b3 = __shfl_sync(0xFFFFFFFFu, t.y, 1);
      if (lane == 0) {
        // r, q and the coefficients; or -1 for statistics that have to be taken in 64 bits, and what the coefficients need.
        const bool again = out_of_range(t.x) || (POST && out_of_range(t.y));
        const float eps = (float)p.eps, r = again ? -1.f : rsqrtf(fmaf(t.x, inv_n, eps)), q = POST && !again ? rsqrtf(fmaf(t.y, inv_n, eps)) : 1.f;
        const float back = r * r * r * (t.z * inv_n);
        sums.row[threadIdx.y] = again ? make_float4(-1.f, t.z, t.w, 0.f) : make_float4(r, q, back, q * q * q * ((t.w + r * b2 - back * b3) * inv_n));
        if (again) { sums.part[first_warp][0] = b2; sums.part[first_warp][1] = b3; }
      }
    }
    group_sync();
    float4 c = sums.row[threadIdx.y];
    if (c.x < 0.f) {       // of the whole group
      const float b2 = sums.part[first_warp][0], b3 = sums.part[first_warp][1];
      double sx = 0.0, sy = 0.0;
#pragma unroll 1
      for (int i = 0; i < NU; ++i) {
        sx += squares_wide<T>(get(X, i));
        if constexpr (POST) sy += squares_wide<T>(get(Y, i));
      }
      group_sync();
      sx = across_warps(warp_sum(sx), sums.wide[0]);
      sy = across_warps(warp_sum(sy), sums.wide[1]);
      const float r = inverse_root(fma(sx, p.inv_n, p.eps)), q = POST ? inverse_root(fma(sy, p.inv_n, p.eps)) : 1.f;
      const float back = r * r * r * (c.y * inv_n);
      c = make_float4(r, q, back, q * q * q * ((c.z + r * b2 - back * b3) * inv_n));
    }
    // ---- gradients
    const F2 r = f2(c.x), q = f2(c.y), back = f2(-c.z), back2 = f2(-c.w);
    uint8_t* const out_x = row_of(p.dx, row, p.lddx);
    uint8_t* const out_y = BLOCK ? row_of(p.dy, row, p.lddy) : nullptr;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int e = unit_at(i);
      if constexpr (HELD) load_vectors(i);
      if constexpr (SHARED) vectors.get(0, i * TX + tx, vw);
      Unit<T> o;
      F2 g[kUnit / 2];
      {
        const Unit<T> x = get(X, i), dh = get(DH, i), d = get(DX, i);
#pragma unroll
        for (int j = 0; j < kUnit / 2; ++j) {
          const F2 xv = pair(x, j), dv = pair(dh, j);
          g[j] = fma2(r, mul2(dv, vw[j]), fma2(back, xv, pair(d, j)));
          if constexpr (HELD) {
            float a, b;
            mul2(dv, mul2(xv, r)).get(a, b);
            if (e + 2 * j < width) { held[e + 2 * j] += a; held[e + 2 * j + 1] += b; }
          } else {
            cw[i][j] = fma2(dv, mul2(xv, r), cw[i][j]);
          }
          float a, b;
          g[j].get(a, b);
          o.set2(2 * j, a, b);
        }
      }
      put_unit<T, FULL>(out_x + e * E, o, p.cols - e);
      if constexpr (BLOCK) {
        if constexpr (SHARED) vectors.get(1, i * TX + tx, vk);
        const Unit<T> y = get(Y, i);
        Unit<T> gate, og;
        if constexpr (MATRIX) gate = get(G, i);
#pragma unroll
        for (int j = 0; j < kUnit / 2; ++j) {
          const F2 yv = pair(y, j), yn = POST ? mul2(yv, q) : yv;
          F2 gv = g[j], t = mul2(gv, vk[j]);                     // g k wp
          float a, b;
          if constexpr (MATRIX) {
            mul2(t, yn).get(a, b);                               // (vk holds wp scale)
            og.set2(2 * j, a, b);
            const F2 k = pair(gate, j);
            t = mul2(t, k);
            gv = mul2(gv, mul2(k, f2(p.scale)));
          }
          if constexpr (HELD) {
            mul2(gv, yn).get(a, b);
            if (e + 2 * j < width) { held[width + e + 2 * j] += a; held[width + e + 2 * j + 1] += b; }
          } else {
            cs[i][j] = fma2(gv, yn, cs[i][j]);
          }
          if constexpr (POST) t = fma2(q, t, mul2(back2, yv));
          t.get(a, b);
          o.set2(2 * j, a, b);
        }
        put_unit<T, FULL>(out_y + e * E, o, p.cols - e);
        if constexpr (MATRIX)
          if (each_row(p.dgate)) put_unit<T, FULL>(row_of(p.dgate, row, p.lddg) + e * E, og, p.cols - e);
      }
    }
    if constexpr (!HELD) {
      __syncwarp();
      issue(row + p.stages * step, at);
    }
    if (++stage == p.stages) stage = 0;
  }
  // ---- this block's column sums (planes of four elements one slot more apart than they have units, for the banks)
  const SharedVectors columns = {sm100::smem_u32(slots), (uint32_t)(width / kUnit + 1) * 16u};
  wait_copies(0);
  __syncthreads();
  if constexpr (!HELD) {
    for (int t = 0; t < (int)blockDim.y; ++t) {
      if ((int)threadIdx.y == t) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          if (unit_at(i) >= p.cols) continue;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            F2* const v = which ? cs[i] : cw[i];
            if (t > 0) {
              F2 before[kUnit / 2];
              columns.get(which, i * TX + tx, before);
#pragma unroll
              for (int j = 0; j < kUnit / 2; ++j) v[j] = add2(before[j], v[j]);
            }
            F2 sum[kUnit / 2];
#pragma unroll
            for (int j = 0; j < kUnit / 2; ++j) sum[j] = v[j];
            columns.put(which, i * TX + tx, sum);
          }
        }
      }
      __syncthreads();
    }
  }
  float* const out = p.parts + (int64_t)blockIdx.x * 2 * p.cols;
  const int all = TX * (int)blockDim.y, me = (int)threadIdx.y * TX + tx;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    for (int q = me; 4 * q < p.cols; q += all) {
      float f[4];
      if constexpr (HELD) {
#pragma unroll
        for (int l = 0; l < 4; ++l) f[l] = held[which * width + 4 * q + l];
      } else {
        F2 a, b;
        columns.get(which, q >> 2, q & 3, a, b);
        a.get(f[0], f[1]);
        b.get(f[2], f[3]);
      }
#pragma unroll
      for (int l = 0; l < 4; ++l)
        if (4 * q + l < p.cols) out[which * p.cols + 4 * q + l] = f[l];
    }
  }
}

struct ColumnParams {
  const float* parts;
  float* dw;
  float* dp;
  float* dg;
  const void* wp;
  const void* gate;
  int32_t param_type, blocks, cols;
  int32_t matrix;
  float scale;
};
// Sums of the blocks' parts: 32 columns per block, 8 slices of the parts; then what the columns of dpost and dgate share.
__global__ void __launch_bounds__(256) residual_norm_columns_kernel(const __grid_constant__ ColumnParams p) {
  __shared__ float slice[8][33];
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const bool second = blockIdx.y == 1;
  if (second ? !p.dp && !p.dg : !p.dw) return;
  const int c = (int)blockIdx.x * 32 + (int)threadIdx.x;
  float s = 0.f;
  if (c < p.cols) {
    const float* const at = p.parts + (int64_t)blockIdx.y * p.cols + c;
#pragma unroll 8
    for (int i = (int)threadIdx.y; i < p.blocks; i += 8) s += at[(int64_t)i * 2 * p.cols];
  }
  slice[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < p.cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += slice[i][threadIdx.x];
    if (!second) {
      p.dw[c] = s;
    } else {
      if (p.dp) p.dp[c] = p.matrix ? s : s * (p.gate ? load_as_f32(p.gate, p.param_type, c) * p.scale : p.scale);
      if (p.dg) p.dg[c] = s * ((p.wp ? load_as_f32(p.wp, p.param_type, c) : 1.f) * p.scale);
    }
  }
}

// Units to a thread: two for 16-bit elements and more rows than SMs.
int back_units(int type, int64_t rows) { return type != GEMM_TYPE_FP32 && rows > 148 ? 2 : 1; }
// `bytes`: a unit's stretches of a warp in all matrices.
Shape back_shape(int type, int64_t rows, int64_t cols, int bytes) {
  const int units = (int)((cols + kUnit - 1) / kUnit);
  if (units > kMaxThreads) {
    Shape s;
    s.tx = kMaxThreads; s.ty = 1; s.stages = 0;
    s.blocks = (int)(rows < 148 ? rows : 148);
    s.smem = (size_t)units * kUnit * 8;
    return s;
  }
  const int nu = back_units(type, rows), vectors = nu == 2 ? ((units + 1) / 2 + 31) / 32 * 32 * 2 * kUnit * 8 : 0;
  return shape_of(rows, units, nu, nu * bytes, kMaxThreads, vectors);
}
// No call has more blocks: with two units there is one to an SM, with one (where rows ahead never limit them) they go by the sizes.
int64_t most_blocks(int64_t rows, int64_t cols) {
  const int64_t two = rows < 148 ? rows : 148, a = back_shape(GEMM_TYPE_FP32, rows, cols, 1).blocks;
  return a > two ? a : two;
}

template <typename T, int KIND>
cudaError_t launch_backward(BackParams p, const Shape& s, bool wide, cudaStream_t st) {
  constexpr bool FP32 = sizeof(T) == 4;
  const int nu = back_units(FP32 ? GEMM_TYPE_FP32 : GEMM_TYPE_BF16, p.rows);
  wide = wide && all_full((p.cols + kUnit - 1) / kUnit, p.cols, nu);
  void (*fn)(BackParams);
  if (p.cols > kMaxThreads * kUnit) {
    fn = residual_norm_backward_kernel<T, 2, true, false, KIND>;
  } else if (nu == 2) {
    fn = wide ? residual_norm_backward_kernel<T, FP32 ? 1 : 2, false, true, KIND> : residual_norm_backward_kernel<T, FP32 ? 1 : 2, false, false, KIND>;
  } else {
    fn = FP32 && wide ? residual_norm_backward_kernel<T, 1, false, FP32, KIND> : residual_norm_backward_kernel<T, 1, false, false, KIND>;
  }
  p.stages = s.stages;
  if (s.stages < 1 && p.cols <= kMaxThreads * kUnit) return cudaErrorInvalidValue;
  const int units = (p.cols + kUnit - 1) / kUnit, vectors = nu == 2 && units <= kMaxThreads ? s.tx * 2 * kUnit * 8 : 0;
  p.vectors_at = (int32_t)s.smem;
  size_t smem = s.smem + vectors;
  const size_t sums = (size_t)(units + 1) * kUnit * 8;  // the column sums lie over it all in the end
  if (smem < sums) smem = sums;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (e != cudaSuccess) return e;
  return launch_overlapped(fn, dim3((unsigned)s.blocks), dim3((unsigned)s.tx, (unsigned)s.ty), smem, 1, st, p);
}
template <typename T>
cudaError_t launch_backward(const BackParams& p, const Shape& s, bool wide, cudaStream_t st) {
  if (!p.in[3]) return launch_backward<T, 0>(p, s, wide, st);
  if (!p.in[4]) return p.wp ? launch_backward<T, 2>(p, s, wide, st) : launch_backward<T, 1>(p, s, wide, st);
  return p.wp ? launch_backward<T, 4>(p, s, wide, st) : launch_backward<T, 3>(p, s, wide, st);
}

int status_of(cudaError_t err) {
  if (err == cudaSuccess) return GEMM_OK;
  cudaGetLastError();
  return GEMM_ERR_LAUNCH;
}
bool aligned(const void* p, int e) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)e == 0; }

// A matrix operand: absent, or with rows of its own that do not run into one another.
struct Mat {
  const void* p;
  int64_t ld;
};

}  // namespace

extern "C" int gemm_sm100a_residual_norm(const ResidualNormArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(ResidualNormArgs)) return GEMM_ERR_BAD_ARGS;
  if (!type_ok(a->type) || a->rows < 0 || a->cols < 1 || a->cols > kMaxCols || a->rows > INT32_MAX / 2) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->param_type != a->type && a->param_type != GEMM_TYPE_FP32) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->block != 0 && !fp4op::block_ok(a->block)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!(a->eps >= 0.0)) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->rows == 0) return GEMM_OK;
  if (!a->x || (a->y != nullptr) != (a->x_out != nullptr) || (!a->y && (a->post_weight || a->gate))) return GEMM_ERR_BAD_ARGS;
  if (a->block ? !a->values || !a->scales || !a->row_scale || a->h : !a->h) return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->type), pe = type_bytes(a->param_type);
  const bool matrix = a->gate && a->ldg != 0;
  if (a->ldx < a->cols || (a->y && (a->ldy < a->cols || a->ldo < a->cols)) || (a->h && a->ldh < a->cols) || (matrix && a->ldg < a->cols))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!aligned(a->x, e) || !aligned(a->y, e) || !aligned(a->x_out, e) || !aligned(a->h, e) || !aligned(a->weight, pe) ||
      !aligned(a->post_weight, pe) || !aligned(a->gate, matrix ? e : pe))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->block && (a->ldv < (a->cols + 1) / 2 || a->ldv % 16 != 0 || !aligned(a->values, 16) || !aligned(a->scales, 16) || !aligned(a->row_scale, 4)))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  auto apart = [&](const void* p, int64_t ldp, const void* o, int64_t ldo) {
    return !p || !o || !rows_meet(p, ldp * e, a->cols * e, o, ldo * e, a->cols * e, a->rows);
  };
  if (a->x_out && (!in_place_or_apart(a->x, a->ldx, a->x_out, a->ldo, a->rows, a->cols, e) ||
                   !in_place_or_apart(a->y, a->ldy, a->x_out, a->ldo, a->rows, a->cols, e) || (matrix && !apart(a->gate, a->ldg, a->x_out, a->ldo))))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!apart(a->x, a->ldx, a->h, a->ldh) || !apart(a->y, a->ldy, a->h, a->ldh) || !apart(a->x_out, a->ldo, a->h, a->ldh) ||
      (matrix && !apart(a->gate, a->ldg, a->h, a->ldh)))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const uint8_t*>(a->x); p.ldx = a->ldx * e; p.y = static_cast<const uint8_t*>(a->y); p.ldy = a->ldy * e;
  p.xo = static_cast<uint8_t*>(a->x_out); p.ldo = a->ldo * e; p.h = static_cast<uint8_t*>(a->h); p.ldh = a->ldh * e;
  p.w = a->weight; p.wp = a->post_weight; p.gate = static_cast<const uint8_t*>(a->gate); p.ldg = matrix ? a->ldg * e : 0;
  p.rows = a->rows; p.cols = (int32_t)a->cols; p.scale = a->scale; p.eps = a->eps; p.inv_n = 1.0 / (double)a->cols;
  p.param32 = a->param_type == GEMM_TYPE_FP32;
  p.values = static_cast<uint8_t*>(a->values); p.ldv = a->ldv; p.scales = static_cast<uint8_t*>(a->scales); p.row_scale = a->row_scale;
  p.tiles = a->block ? fp4op::scale_tiles(a->cols, a->block) : 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->block ? a->values : a->h);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  p.block = a->block;
  return status_of(a->type == GEMM_TYPE_BF16 ? launch_forward<__nv_bfloat16>(p, st)
                 : a->type == GEMM_TYPE_FP16 ? launch_forward<__half>(p, st) : launch_forward<float>(p, st));
}

extern "C" int64_t gemm_sm100a_residual_norm_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1 || cols > kMaxCols || rows > INT32_MAX / 2) return -1;
  if (rows == 0) return 0;
  return most_blocks(rows, cols) * 2 * cols * 4;
}

extern "C" int gemm_sm100a_residual_norm_backward(const ResidualNormBackwardArgs* a, void* stream) {
  if (!a || a->struct_size != sizeof(ResidualNormBackwardArgs)) return GEMM_ERR_BAD_ARGS;
  if (!type_ok(a->type) || a->rows < 0 || a->cols < 1 || a->cols > kMaxCols || a->rows > INT32_MAX / 2) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (a->param_type != a->type && a->param_type != GEMM_TYPE_FP32) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!(a->eps >= 0.0)) return GEMM_ERR_CANNOT_IMPLEMENT;
  const bool matrix = a->gate && a->ldg != 0;
  if (a->rows > 0 && ((!a->weight && a->dweight) || (!a->post_weight && a->dpost_weight) || (!a->gate && a->dgate) ||
                      (!a->y && (a->dy || a->post_weight || a->gate))))
    return GEMM_ERR_BAD_ARGS;
  const int e = type_bytes(a->type), pe = type_bytes(a->param_type);
  if (!aligned(a->dweight, 4) || !aligned(a->dpost_weight, 4) || !aligned(a->dgate, matrix ? e : 4)) return GEMM_ERR_CANNOT_IMPLEMENT;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  float* const sums[3] = {a->dweight, a->dpost_weight, matrix ? nullptr : static_cast<float*>(a->dgate)};
  const bool any = sums[0] || sums[1] || sums[2];
  if (a->rows == 0) {
    for (float* s : sums) {
      if (!s) continue;
      PointerDeviceGuard guard(s);
      if (!guard.ok) return GEMM_ERR_LAUNCH;
      const int rc = status_of(cudaMemsetAsync(s, 0, (size_t)a->cols * 4, st));
      if (rc != GEMM_OK) return rc;
    }
    return GEMM_OK;
  }
  if (!a->dh || !a->x_out || !a->dx || (a->y && !a->dy) || !a->workspace) return GEMM_ERR_BAD_ARGS;
  const Mat ins[5] = {{a->x_out, a->ldo}, {a->dh, a->lddh}, {a->dx_out, a->lddo}, {a->y, a->ldy}, {matrix ? a->gate : nullptr, a->ldg}};
  const Mat outs[3] = {{a->dx, a->lddx}, {a->dy, a->lddy}, {matrix ? a->dgate : nullptr, a->lddg}};
  for (const Mat& m : ins)
    if (m.p && (m.ld < a->cols || !aligned(m.p, e))) return GEMM_ERR_CANNOT_IMPLEMENT;
  for (const Mat& m : outs)
    if (m.p && (m.ld < a->cols || !aligned(m.p, e))) return GEMM_ERR_CANNOT_IMPLEMENT;
  if (!aligned(a->weight, pe) || !aligned(a->post_weight, pe) || (a->gate && !matrix && !aligned(a->gate, pe)) || !aligned(a->workspace, 16))
    return GEMM_ERR_CANNOT_IMPLEMENT;
  // The row is read again after the first stores of its gradients: outputs lie over nothing.
  for (int i = 0; i < 3; ++i) {
    for (const Mat& m : ins)
      if (outs[i].p && m.p && rows_meet(m.p, m.ld * e, a->cols * e, outs[i].p, outs[i].ld * e, a->cols * e, a->rows)) return GEMM_ERR_CANNOT_IMPLEMENT;
    for (int j = 0; j < i; ++j)
      if (outs[i].p && outs[j].p && rows_meet(outs[j].p, outs[j].ld * e, a->cols * e, outs[i].p, outs[i].ld * e, a->cols * e, a->rows))
        return GEMM_ERR_CANNOT_IMPLEMENT;
  }
  bool wide = true;
  for (const Mat& m : ins) wide &= !m.p || rows_16b(m.p, m.ld, e);
  for (const Mat& m : outs) wide &= !m.p || rows_16b(m.p, m.ld, e);
  const uint32_t place = place_bytes(e, wide);
  const Shape s = back_shape(a->type, a->rows, a->cols, ((a->y ? 4 : 3) + (matrix ? 1 : 0)) * (int)place);
  if (a->workspace_bytes < (int64_t)s.blocks * 2 * a->cols * 4) return GEMM_ERR_BAD_ARGS;
  BackParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < 5; ++i) {
    p.in[i] = static_cast<const uint8_t*>(ins[i].p);
    p.ld[i] = ins[i].ld * e;
  }
  p.w = a->weight; p.wp = a->post_weight; p.gate = matrix ? nullptr : a->gate;
  p.dx = static_cast<uint8_t*>(a->dx); p.lddx = a->lddx * e; p.dy = static_cast<uint8_t*>(a->dy); p.lddy = a->lddy * e;
  p.dgate = matrix ? static_cast<uint8_t*>(a->dgate) : nullptr; p.lddg = a->lddg * e;
  p.parts = static_cast<float*>(a->workspace);
  p.rows = a->rows; p.cols = (int32_t)a->cols; p.scale = a->scale; p.eps = a->eps; p.inv_n = 1.0 / (double)a->cols;
  p.param32 = a->param_type == GEMM_TYPE_FP32;
  p.place = place;
  PointerDeviceGuard guard(a->dx);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  cudaError_t err = a->type == GEMM_TYPE_BF16 ? launch_backward<__nv_bfloat16>(p, s, wide, st)
                  : a->type == GEMM_TYPE_FP16 ? launch_backward<__half>(p, s, wide, st) : launch_backward<float>(p, s, wide, st);
  if (err == cudaSuccess && any) {
    ColumnParams c;
    memset(&c, 0, sizeof(c));
    c.parts = p.parts;
    c.dw = sums[0]; c.dp = sums[1]; c.dg = sums[2];
    c.wp = a->post_weight; c.gate = matrix ? nullptr : a->gate;
    c.param_type = a->param_type; c.blocks = s.blocks; c.cols = p.cols;
    c.matrix = matrix; c.scale = a->scale;
    err = launch_overlapped(residual_norm_columns_kernel, dim3((unsigned)((p.cols + 31) / 32), 2), dim3(32, 8), 0, 1, st, c);
  }
  return status_of(err);
}
