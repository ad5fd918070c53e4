// residual_norm_backward.cu -- gradients of the residual stream around a block (residual_norm.cu).  Bound by the bytes of
// six matrices.
//
// With c columns, dn = dh w, k = gate scale, P = k wp y, r = r(x'), q = r(y), n = x' r, m = y q:
//   g  = dx' + r (dn - a n)                a = mean(dn n) = r (sum dn x') / c
//   dy = q (k wp g - b m)                  b = q mean(P g) = q (sum P g) / c
//   sum P g = sum P dx' + r (sum P dn - a (r sum P x'))
// (with n and m, whatever the rows' magnitude; r^3 and q^3 would leave fp32's range long before the gradients do), so that all row sums (with those of x'^2 and y^2) come from one pass and one exchange, and no statistics are
// kept from the forward call.  The sums over rows (dw, dwp, dgate) stay with the threads of a block, which walks down the
// matrix; the blocks' parts go through a workspace to a second kernel that adds them in order.
//
// Measured on B200: 16384 x 8192 bf16 with gate and fp32 vectors 327 to 347 us a call (4.6 to 4.9 of the 6.55 TB/s that a copy
// reaches); bound by latency: the column sums' registers and the vectors leave room for two groups of 8 warps and one row
// each, the next row is asked for after the second pass of the one before, and between its two barriers a group's first warp
// works alone (issue slots 48 % busy).  With a gate matrix 412, fp32 694; 4096 x 8192 rows of zeros 99.
// 333 x 1001 fp32 with a gate matrix 13 us, of which the host's call is 9.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "device_guard.cuh"
#include "gemm_sm100a.h"
#include "residual_norm.cuh"

namespace {

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
  float low, high;                       // sums of squares that fp32 holds, with what is made of them
  int32_t stages;
  uint32_t place;
  int32_t param32;
  int32_t vectors_at;
};

// Row sums: 0 x^2, 1 y^2, 2 dn x, 3 P dx', 4 P dn, 5 P x.
struct BackSums {
  float part[kMaxThreads / 32][8];
  double wide[2][kMaxThreads / 32];
  float4 row[kMaxThreads / 32];  // r, q, a and b, one row to a group
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
  constexpr int E = (int)sizeof(T);
  constexpr bool BLOCK = KIND > 0, POST = KIND == 2 || KIND == 4, MATRIX = KIND > 2, SHARED = NU == 2 && !HELD;
  enum { X, DH, DX, Y, G };
  const int tx = threadIdx.x, TX = blockDim.x;
  const int width = (p.cols + kUnit - 1) / kUnit * kUnit;
  const uint32_t per_stage = (uint32_t)((BLOCK ? 4 : 3) + (MATRIX ? 1 : 0)) * NU * p.place;
  const uint32_t mine = sm100::smem_u32(slots) + (uint32_t)((int)threadIdx.y * (TX >> 5) + (tx >> 5)) * (uint32_t)p.stages * per_stage;
  auto unit_at = [&](int i) { return (i * TX + tx) * kUnit; };
  // Column sums in shared memory (HELD, and in the end): planes of four elements, one slot more apart than there are units, for
  // the banks.
  const SharedVectors columns = {sm100::smem_u32(slots), (uint32_t)(width / kUnit + 1) * 16u};
  if constexpr (HELD) {
    const F2 none[kUnit / 2] = {f2(0.f), f2(0.f), f2(0.f), f2(0.f), f2(0.f), f2(0.f), f2(0.f), f2(0.f)};
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (unit_at(i) < p.cols) {       // a unit's sums are its thread's own
        columns.put(0, i * TX + tx, none);
        columns.put(1, i * TX + tx, none);
      }
  }
  auto add_held = [&](int which, int i, F2 (&v)[kUnit / 2]) {
    if (unit_at(i) >= p.cols) return;
    F2 before[kUnit / 2];
    columns.get(which, i * TX + tx, before);
#pragma unroll
    for (int j = 0; j < kUnit / 2; ++j) v[j] = add2(before[j], v[j]);
    columns.put(which, i * TX + tx, v);
  };
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
      const float s4 = __shfl_sync(0xFFFFFFFFu, t.x, 1), s5 = __shfl_sync(0xFFFFFFFFu, t.y, 1);
      if (lane == 0) {
        // r, q, a and b; or -1 for sums that have to be taken in 64 bits.
        const float eps = (float)p.eps, r = rsqrtf(fmaf(t.x, inv_n, eps)), q = POST ? rsqrtf(fmaf(t.y, inv_n, eps)) : 1.f;
        const float a = r * t.z * inv_n, b = q * ((t.w + r * (s4 - a * (r * s5))) * inv_n);
        const bool held = t.x > p.low && t.x < p.high && (!POST || (t.y > p.low && t.y < p.high)) && fabsf(a) + fabsf(b) < __int_as_float(0x7F800000);
        sums.row[threadIdx.y] = make_float4(held ? r : -1.f, q, a, b);
      }
    }
    group_sync();
    float4 c = sums.row[threadIdx.y];
    if (c.x < 0.f) {       // of the whole group
      double w[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
      auto element = [&](int m, int col) { return (double)to_f32(reinterpret_cast<const T*>(p.in[m] + row * p.ld[m])[col]); };
      auto param = [&](const void* v, int col) {
        return !v ? 1.f : sizeof(T) == 4 || p.param32 ? static_cast<const float*>(v)[col] : to_f32(static_cast<const T*>(v)[col]);
      };
#pragma unroll 1
      for (int col = tx; col < p.cols; col += TX) {
        const double xv = element(X, col), dn = element(DH, col) * param(p.w, col);
        w[0] = fma(xv, xv, w[0]);
        w[2] = fma(dn, xv, w[2]);
        if constexpr (POST) {
          const double yv = element(Y, col), f = yv * param(p.wp, col) * (MATRIX ? element(G, col) : (double)param(p.gate, col)) * p.scale;
          w[1] = fma(yv, yv, w[1]);
          if (p.in[DX]) w[3] = fma(f, element(DX, col), w[3]);
          w[4] = fma(f, dn, w[4]);
          w[5] = fma(f, xv, w[5]);
        }
      }
#pragma unroll
      for (int k = 0; k < 6; ++k)
        if (POST || k == 0 || k == 2) w[k] = group_sum(w[k], sums.wide[POST ? k & 1 : k / 2]);
      const double r = 1.0 / sqrt(fma(w[0], p.inv_n, p.eps)), q = POST ? 1.0 / sqrt(fma(w[1], p.inv_n, p.eps)) : 1.0;
      const double a = r * w[2] * p.inv_n;
      c = make_float4((float)r, (float)q, (float)a, (float)(q * ((w[3] + r * (w[4] - a * (r * w[5]))) * p.inv_n)));
    }
    // ---- gradients
    const F2 r = f2(c.x), q = f2(c.y), minus_a = f2(-c.z), minus_b = f2(-c.w);
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
          const F2 n = mul2(pair(x, j), r), dv = pair(dh, j);
          g[j] = fma2(r, fma2(minus_a, n, mul2(dv, vw[j])), pair(d, j));
          if constexpr (HELD) cw[i][j] = mul2(dv, n);
          else cw[i][j] = fma2(dv, n, cw[i][j]);
          float a, b;
          g[j].get(a, b);
          o.set2(2 * j, a, b);
        }
      }
      if constexpr (HELD) add_held(0, i, cw[i]);
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
          if constexpr (HELD) cs[i][j] = mul2(gv, yn);
          else cs[i][j] = fma2(gv, yn, cs[i][j]);
          if constexpr (POST) t = mul2(q, fma2(minus_b, yn, t));
          t.get(a, b);
          o.set2(2 * j, a, b);
        }
        if constexpr (HELD) add_held(1, i, cs[i]);
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
  // ---- this block's column sums
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
      F2 a, b;
      columns.get(which, q >> 2, q & 3, a, b);
      a.get(f[0], f[1]);
      b.get(f[2], f[3]);
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
    s.tx = ((units + 1) / 2 + 31) / 32 * 32; s.ty = 1; s.stages = 0;
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

// A matrix operand, or none.
struct Mat {
  const void* p;
  int64_t ld;
};

}  // namespace

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
  // Sums of squares below 1e20 leave room for products with gradients. Small ones lose what eps does not outweigh.
  p.low = a->eps < 1e-12 ? 1e-20f : -1.f;
  p.high = a->eps < 1e30 ? 1e20f : 0.f;
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
