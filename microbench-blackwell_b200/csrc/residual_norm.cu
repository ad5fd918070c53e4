// residual_norm.cu -- the residual stream around a block: the norm after it, its gate and scale, the stream's
// update and the norm before the next block.  Bound by the bytes of the rows: four matrices, or three and a quarter where
// the result becomes a 4-bit operand.
//
//   z = y r(y) wp,  x' = x + (gate scale) z,  h = x' r(x') w,  r(v) = 1 / sqrt(mean(v^2) + eps)
//
// Measured on B200: 16384 x 8192 bf16 with gate and fp32 vectors 172 to 200 us a call (5.4 to 6.2 of the 6.55 TB/s that a copy
// reaches: the same build gives either, as the memory serves four streams), with a gate matrix 236, from fp32 398 us; into a 4-bit
// operand 223 us, bound by issue slots (67 % busy); one row 4.8 and 6.9 us a call.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "fp4_common.cuh"
#include "gemm_sm100a.h"
#include "residual_norm.cuh"

namespace {

constexpr int kManyThreads = 768;          // of a block of many rows
template <typename T, int KIND>
constexpr int many_threads() { return sizeof(T) == 2 && KIND != 3 ? kManyThreads : kMaxThreads; }

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
  int32_t gate_vector;         // gate scale is a vector in shared memory (KIND 3: its first half is); else it is scale (KIND 3: in the caches)
};

// NU units to a thread, blockDim.x units apart.
//  Few rows (NU 1): the vectors stay in registers.
//  Many rows (NU 2, which halves what the statistics cost per element) of 16-bit elements: the vectors lie in shared memory as w, wp and gate
//    scale, in fp32, where all groups of the block read them, and three groups of 8192-element rows hide one another's
//    barriers (292 us; with the vectors in the registers of one group 353).  Rows of fp32 read them from the caches each time.
// KIND 0: no y; 1: y; 2: y and a gate matrix; 3: y and a gate vector of 16-bit rows that shared memory has no room for (more than
// 14336 elements, 13312 off 16-byte boundaries): each thread's second unit of it, and where there is no room for half a vector (beyond
// 15360 off 16-byte boundaries) its first, is read from the caches for each row, before the barriers of the first statistics
// (4096 x 16384 with an fp32 gate 159 us, 108 with one product of wp and gate made before, which rounds in another order
// and may leave fp32's range where z does not).
// (What can be absent from call to call is decided here where the compiler would otherwise make a copy of the loop for each
// case, with the registers of all.)
template <typename T, bool FOUR, int NU, bool FULL, int KIND>
__global__ void __launch_bounds__(NU == 2 ? many_threads<T, KIND>() : kMaxThreads, 1) residual_norm_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ double part[2][kManyThreads / 32];
  __shared__ WarpSum part32[2][kManyThreads / 32];
  __shared__ uint32_t warp_max[kManyThreads / 32];
  constexpr int E = (int)sizeof(T);
  constexpr bool KEEP = NU == 1, SHARED = NU == 2 && E == 2, BLOCK = KIND > 0, MATRIX = KIND == 2, CACHED = KIND == 3;
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

  F2 vw[kUnit / 2], vp[kUnit / 2], vk[kUnit / 2];      // w, wp, gate scale
  auto load_w = [&](int i) { load_params<T>(p.w, p.param32, e[i], n[i], vw); };
  auto load_k = [&](int i) {
    load_params<T>(p.wp, p.param32, e[i], n[i], vp);
    if constexpr (!MATRIX) {
      load_params<T>(p.gate, p.param32, e[i], n[i], vk);
#pragma unroll
      for (int j = 0; j < kUnit / 2; ++j) vk[j] = mul2(vk[j], f2(p.scale));
    }
  };
  const SharedVectors vectors = {sm100::smem_u32(slots) + (uint32_t)p.vectors_at, (uint32_t)(NU * TX) * 16u};
  const SharedVectors half_gate = {vectors.base + 8u * vectors.per_chunk, (uint32_t)TX * 16u};
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
          if (CACHED && i == 0 && p.gate_vector) half_gate.put(0, tx, vk);
          vectors.put(1, i * TX + tx, vp);
          if (!MATRIX && !CACHED && p.gate_vector) vectors.put(2, i * TX + tx, vk);
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
      s = group_sum(s, at);
    } else {
      float hi, lo;
      squares<T, NU>(v, hi, lo);
      s = group_sum_parts(hi, lo, part32[flip]);
      if (out_of_range((float)s)) {
        group_sync();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < NU; ++i) s += squares_wide<T>(v[i]);
        s = group_sum(s, at);
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
      F2 late[CACHED ? NU : 1][kUnit / 2];
      if constexpr (CACHED) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
          if (i > 0 || !each_row(p.gate_vector)) load_params<T>(p.gate, p.param32, e[i], n[i], late[i]);
      }
      const F2 q = f2(p.wp ? inverse_rms(y) : 1.f);
#pragma unroll
      for (int i = 0; i < NU; ++i) forget(y[i]);
      uint8_t* const out = row_of(p.xo, row, p.ldo);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (!KEEP && !SHARED) load_k(i);
        const bool gated = SHARED && !MATRIX && !CACHED && each_row(p.gate_vector);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          F2 w[2] = {vp[2 * c], vp[2 * c + 1]}, k[2] = {vk[2 * c], vk[2 * c + 1]};
          if (SHARED) {
            vectors.get(1, i * TX + tx, c, w[0], w[1]);
            if constexpr (CACHED) {
              if (i == 0 && each_row(p.gate_vector)) {
                half_gate.get(0, tx, c, k[0], k[1]);
              } else {
                k[0] = mul2(late[i][2 * c], f2(p.scale));
                k[1] = mul2(late[i][2 * c + 1], f2(p.scale));
              }
            } else if (!MATRIX) {
              k[0] = k[1] = f2(p.scale);
              if (gated) vectors.get(2, i * TX + tx, c, k[0], k[1]);
            }
          }
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            const int j = 2 * c + l;
            F2 z = mul2(mul2(pair(y[i], j), q), w[l]);
            if (MATRIX) k[l] = mul2(pair(gate[i], j), f2(p.scale));
            // (A product and a sum of pairs become one multiply-add, whatever their rounding modes say; two sums do not.)
            float a, b;
            mul2(z, k[l]).get(a, b);
            x[i].set2(2 * j, __fadd_rn(x[i].get(2 * j), a), __fadd_rn(x[i].get(2 * j + 1), b));
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
  const int tx = ((units + NU - 1) / NU + 31) / 32 * 32, vector = SHARED ? tx * NU * kUnit * 4 : 0;
  if constexpr (SHARED && KIND == 1)
    if (p.gate && 3 * vector + two * (tx / 32) > kSmemLimit) return launch_forward<T, FOUR, NU, FULL, 3>(p0, st);
  p.gate_vector = KIND == 3 ? 2 * vector + vector / 2 + two * (tx / 32) <= kSmemLimit : KIND == 1 && p.gate;
  const int vectors = KIND == 0 ? vector : 2 * vector + (p.gate_vector ? vector / (KIND == 3 ? 2 : 1) : 0);
  // A gate matrix is not copied ahead where there is no room for it (16-bit rows of more than 15360 elements off 16-byte boundaries).
  p.gate_ahead = KIND == 2 && vectors + three * (tx / 32) <= kSmemLimit;
  const Shape s = shape_of(p.rows, units, NU, p.gate_ahead ? three : two, NU == 2 ? many_threads<T, KIND>() : kMaxThreads, vectors);
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
