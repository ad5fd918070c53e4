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
#include "row_vec.cuh"
#include "sm100_ptx.cuh"

using namespace int8op;
using rowvec::kUnit;
using rowvec::Unit;

namespace {

constexpr int kMaxCols = 16384;
constexpr int kMaxThreads = 512;

// Squares of a unit.  Those of 16-bit elements are exact in fp32 and added there, 16 at a time; where that leaves
// fp32's range (or comes near its end) the row is summed again in 64 bits.
template <typename T>
__device__ __forceinline__ double squares(const Unit<T>& u, bool wide) {
  if (sizeof(T) == 4 || wide) {
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) s = fma((double)u.get(j), (double)u.get(j), s);
    return s;
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < kUnit; ++j) s = fmaf(u.get(j), u.get(j), s);
  return (double)s;
}
__device__ __forceinline__ bool out_of_range(double s) { return !(s > 1e-30 && s < 1e38); }

// 1 / sqrt(v), rounded to fp32 from an error of 2^-43 or less.
__device__ __forceinline__ float inverse_root(double v) {
  if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
  const double r = (double)rsqrtf((float)v);
  return (float)fma(0.5 * r, fma(-v * r, r, 1.0), r);
}

// Row sums of blockDim.x threads (whole warps); blockDim.y rows at a time, all threads of the block call.
// `slot` alternates between calls.
struct RowSums {
  double part[2][kMaxThreads / 32];
};
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double row_sum(double v, RowSums& sums, int slot) {
  v = warp_sum(v);
  const int warps = (int)blockDim.x >> 5;
  if (warps == 1) return v;
  const int first = (int)threadIdx.y * warps;
  if ((threadIdx.x & 31u) == 0) sums.part[slot][first + (threadIdx.x >> 5)] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < warps; ++i) s += sums.part[slot][first + i];
  return s;
}

struct NormParams {
  const void* x; int64_t ldx;
  const void* y; int64_t ldy;
  void* xo; int64_t ldo;
  void* h; int64_t ldh;
  const void* w;
  const void* wp;
  const void* gate; int64_t ldg;
  int64_t rows;
  int32_t cols;
  float scale;
  double eps;
  uint8_t* values; int64_t ldv;
  uint8_t* scales;
  float* row_scale;
  int64_t tiles;
};

// Element j of (gate scale), in the order of the definition.
template <typename P>
__device__ __forceinline__ Unit<float> gate_scale(const Unit<P>& g, float scale) {
  Unit<float> k;
#pragma unroll
  for (int j = 0; j < kUnit; ++j) k.w[j] = __float_as_uint(__fmul_rn(g.get(j), scale));
  return k;
}

template <typename T, typename P, int BLOCK, int NU>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ RowSums sums;
  __shared__ uint32_t warp_max[kMaxThreads / 32];
  const int tx = threadIdx.x, TX = blockDim.x;
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const int cols = live ? p.cols : 0;
  const int64_t r0 = live ? row : 0;
  Unit<T> x[NU], y[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int e = (i * TX + tx) * kUnit;
    x[i] = rowvec::load_unit<T>(static_cast<const T*>(p.x) + r0 * p.ldx + e, cols - e);
    if (p.y) y[i] = rowvec::load_unit<T>(static_cast<const T*>(p.y) + r0 * p.ldy + e, cols - e);
  }
  auto inverse_rms = [&](const Unit<T> (&v)[NU], int slot) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < NU; ++i) s += squares<T>(v[i], false);
    s = row_sum(s, sums, slot);
    if constexpr (sizeof(T) == 2) {
      // All rows of the block go this way, or none.
      if (blockDim.y == 1 ? out_of_range(s) : __syncthreads_or(out_of_range(s))) {
        __syncthreads();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < NU; ++i) s += squares<T>(v[i], true);
        s = row_sum(s, sums, slot);
      }
    }
    return inverse_root(s / p.cols + p.eps);
  };
  if (p.y) {
    const float q = p.wp ? inverse_rms(y, 0) : 1.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int e = (i * TX + tx) * kUnit;
      float z[kUnit];
#pragma unroll
      for (int j = 0; j < kUnit; ++j) z[j] = y[i].get(j);
      if (p.wp) {
        const Unit<P> wp = rowvec::load_unit<P, rowvec::kKeep>(static_cast<const P*>(p.wp) + e, cols - e);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) z[j] = __fmul_rn(__fmul_rn(z[j], q), wp.get(j));
      }
      if (!p.gate) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) z[j] = __fmul_rn(z[j], p.scale);
      } else {
        const Unit<float> k = p.ldg ? gate_scale(rowvec::load_unit<T>(static_cast<const T*>(p.gate) + r0 * p.ldg + e, cols - e), p.scale)
                                    : gate_scale(rowvec::load_unit<P, rowvec::kKeep>(static_cast<const P*>(p.gate) + e, cols - e), p.scale);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) z[j] = __fmul_rn(z[j], k.get(j));
      }
#pragma unroll
      for (int j = 0; j < kUnit; j += 2) x[i].set2(j, __fadd_rn(x[i].get(j), z[j]), __fadd_rn(x[i].get(j + 1), z[j + 1]));
      rowvec::store_unit<T>(static_cast<T*>(p.xo) + r0 * p.ldo + e, x[i], cols - e);
    }
  }
  const float r = inverse_rms(x, 1);
  // h of a unit, in fp32.
  auto norm = [&](int i, float (&h)[kUnit]) {
    const int e = (i * TX + tx) * kUnit;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) h[j] = __fmul_rn(x[i].get(j), r);
    if (p.w) {
      const Unit<P> w = rowvec::load_unit<P, rowvec::kKeep>(static_cast<const P*>(p.w) + e, cols - e);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) h[j] = __fmul_rn(h[j], w.get(j));
    }
  };
  if constexpr (BLOCK == 0) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int e = (i * TX + tx) * kUnit;
      float h[kUnit];
      norm(i, h);
      Unit<T> o;
#pragma unroll
      for (int j = 0; j < kUnit; j += 2) o.set2(j, h[j], h[j + 1]);
      rowvec::store_unit<T>(static_cast<T*>(p.h) + r0 * p.ldh + e, o, cols - e);
    }
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      float h[kUnit];
      norm(i, h);
#pragma unroll
      for (int j = 0; j < kUnit; ++j)
        if ((i * TX + tx) * kUnit + j < cols) top = max(top, __float_as_uint(h[j]) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (TX > 32) {
      const int first = (int)threadIdx.y * (TX >> 5);
      if ((tx & 31) == 0) warp_max[first + (tx >> 5)] = top;
      __syncthreads();
      top = __reduce_max_sync(0xFFFFFFFFu, (tx & 31) < (TX >> 5) ? warp_max[first + (tx & 31)] : 0u);
    }
    const fp4op::RowScale s = fp4op::row_scale(top);
    if (live && tx == 0) p.row_scale[row] = s.scale;
    const int units = (int)p.tiles * 4 * (BLOCK / 16);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int unit = i * TX + tx;
      if ((unit & ~31) >= units) break;      // whole warps
      float h[kUnit];
      norm(i, h);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) h[j] = s.up == 0.f || unit * kUnit + j >= cols ? 0.f : h[j] * s.up;
      uint32_t q[2];
      const uint32_t code = fp4op::quantize_unit<BLOCK>(h, q);
      fp4op::store_scale_codes<BLOCK>(p.scales, row, p.tiles, unit, code, live && unit < units);
      const int n = cols - unit * kUnit;
      if (n > 0) fp4op::store_codes(p.values + row * p.ldv + unit * 8, q, n);
    }
  }
}

template <typename T, typename P, int BLOCK, int NU>
cudaError_t launch_forward(const NormParams& p, cudaStream_t st) {
  const int units = BLOCK ? (int)p.tiles * 4 * (BLOCK / 16) : (p.cols + kUnit - 1) / kUnit;
  int tx = ((units + NU - 1) / NU + 31) / 32 * 32;
  const int ty = tx >= 128 ? 1 : 128 / tx;
  return launch_overlapped(residual_norm_kernel<T, P, BLOCK, NU>, dim3((unsigned)((p.rows + ty - 1) / ty)), dim3((unsigned)tx, (unsigned)ty), 0, 1, st, p);
}
template <typename T, typename P, int BLOCK>
cudaError_t launch_forward(const NormParams& p, cudaStream_t st) {
  return p.cols <= kMaxThreads * kUnit / 2 ? launch_forward<T, P, BLOCK, 1>(p, st) : launch_forward<T, P, BLOCK, 2>(p, st);
}
template <typename T, typename P>
cudaError_t launch_forward(const NormParams& p, int block, cudaStream_t st) {
  return block == 0 ? launch_forward<T, P, 0>(p, st) : block == 16 ? launch_forward<T, P, 16>(p, st) : launch_forward<T, P, 32>(p, st);
}

// ----------------------------------------------------------------- backward
struct BackParams {
  const void* dh; int64_t lddh;
  const void* dxo; int64_t lddo;
  const void* xo; int64_t ldo;
  const void* y; int64_t ldy;
  const void* w;
  const void* wp;
  const void* gate; int64_t ldg;
  void* dx; int64_t lddx;
  void* dy; int64_t lddy;
  void* dgate; int64_t lddg;     // matrix; NULL where it is a vector
  float* parts;                  // [CTA][3][cols]: dw, dwp, dgate
  int64_t rows;
  int32_t cols;
  float scale;
  double eps;
};

struct BackSums {
  double squares[2][2][kMaxThreads / 32];
  float4 dots[2][kMaxThreads / 32];
};

// A thread's units lie blockDim.x units apart (one; two for rows of more than 8192 elements, whose column sums then are in
// shared memory: HELD).  The row is read twice, the second time from the caches.
template <typename T, typename P, bool HELD>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_backward_kernel(const __grid_constant__ BackParams p) {
  extern __shared__ float held[];          // [3][cols rounded up to units]: column sums (HELD, and to add those of blockDim.y rows)
  __shared__ BackSums sums;
  const int tx = threadIdx.x, TX = blockDim.x;
  const int width = (p.cols + kUnit - 1) / kUnit * kUnit;
  constexpr int NU = HELD ? 2 : 1;
  float cw[kUnit], cp[kUnit], cg[kUnit];
#pragma unroll
  for (int j = 0; j < kUnit; ++j) cw[j] = cp[j] = cg[j] = 0.f;
  if constexpr (HELD) {
    for (int i = tx; i < 3 * width; i += TX) held[i] = 0.f;
    __syncthreads();
  }
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  const float inv_n = 1.f / (float)p.cols;
  int slot = 0;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  for (int64_t base = (int64_t)blockIdx.x * blockDim.y; base < p.rows; base += step, slot ^= 1) {
    const int64_t row = base + threadIdx.y;
    const bool live = row < p.rows;
    const int cols = live ? p.cols : 0;
    const int64_t r0 = live ? row : 0;
    auto load = [&](const void* m, int64_t ld, int e) { return rowvec::load_unit<T, rowvec::kKeep>(static_cast<const T*>(m) + r0 * ld + e, cols - e); };
    auto param = [&](const void* v, int e) { return rowvec::load_unit<P, rowvec::kKeep>(static_cast<const P*>(v) + e, p.cols - e); };
    // k of a unit: gate scale, or scale alone.
    auto factor = [&](int e) {
      Unit<float> k;
      if (p.gate) return p.ldg ? gate_scale(load(p.gate, p.ldg, e), p.scale) : gate_scale(param(p.gate, e), p.scale);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) k.w[j] = __float_as_uint(p.scale);
      return k;
    };
    // ---- row sums
    double sx = 0.0, sy = 0.0;
    float a = 0.f, b1 = 0.f, b2 = 0.f, b3 = 0.f;
    auto add = [&](int i, bool wide) {
      const int e = (i * TX + tx) * kUnit;
      const Unit<T> x = load(p.xo, p.ldo, e);
      sx += squares<T>(x, wide);
      Unit<T> y;
      if (p.wp) {
        y = load(p.y, p.ldy, e);
        sy += squares<T>(y, wide);
      }
      if (wide) return;
      const Unit<T> dh = load(p.dh, p.lddh, e);
      float dn[kUnit];
#pragma unroll
      for (int j = 0; j < kUnit; ++j) dn[j] = dh.get(j);
      if (p.w) {
        const Unit<P> w = param(p.w, e);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) dn[j] *= w.get(j);
      }
#pragma unroll
      for (int j = 0; j < kUnit; ++j) a = fmaf(dn[j], x.get(j), a);
      if (p.wp) {
        const Unit<float> k = factor(e);
        const Unit<P> wp = param(p.wp, e);
        Unit<T> d;
        if (p.dxo) d = load(p.dxo, p.lddo, e); else d.clear();
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          const float f = k.get(j) * wp.get(j) * y.get(j);
          b1 = fmaf(f, d.get(j), b1);
          b2 = fmaf(f, dn[j], b2);
          b3 = fmaf(f, x.get(j), b3);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < NU; ++i) add(i, false);
    auto exchange = [&](int s, bool dots) {
      const int warps = TX >> 5, first = (int)threadIdx.y * warps, at = first + (tx >> 5);
      sx = warp_sum(sx);
      if (p.wp) sy = warp_sum(sy);
      if (dots) {
        a = warp_sum(a);
        if (p.wp) { b1 = warp_sum(b1); b2 = warp_sum(b2); b3 = warp_sum(b3); }
      }
      if (warps == 1) return;
      if ((tx & 31) == 0) {
        sums.squares[s][0][at] = sx;
        sums.squares[s][1][at] = sy;
        if (dots) sums.dots[s][at] = make_float4(a, b1, b2, b3);
      }
      __syncthreads();
      sx = sy = 0.0;
      if (dots) a = b1 = b2 = b3 = 0.f;
      for (int i = first; i < first + warps; ++i) {
        sx += sums.squares[s][0][i];
        sy += sums.squares[s][1][i];
        if (dots) {
          const float4 d = sums.dots[s][i];
          a += d.x; b1 += d.y; b2 += d.z; b3 += d.w;
        }
      }
    };
    exchange(slot, true);
    if constexpr (sizeof(T) == 2) {
      const bool again = out_of_range(sx) || (p.wp && out_of_range(sy));
      if (blockDim.y == 1 ? again : __syncthreads_or(again)) {
        __syncthreads();
        sx = sy = 0.0;
#pragma unroll
        for (int i = 0; i < NU; ++i) add(i, true);
        exchange(slot, false);
        __syncthreads();
      }
    }
    const float r = inverse_root(sx / p.cols + p.eps);
    const float q = p.wp ? inverse_root(sy / p.cols + p.eps) : 1.f;
    const float back = r * r * r * (a * inv_n);
    const float back2 = q * q * q * ((b1 + r * b2 - back * b3) * inv_n);
    // ---- gradients
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int e = (i * TX + tx) * kUnit;
      const Unit<T> x = load(p.xo, p.ldo, e), dh = load(p.dh, p.lddh, e);
      Unit<T> o;
      float g[kUnit];
      if (p.dxo) {
        const Unit<T> d = load(p.dxo, p.lddo, e);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) g[j] = d.get(j);
      } else {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) g[j] = 0.f;
      }
      float nw[kUnit], np[kUnit], ng[kUnit];         // this row's parts of the column sums
      if (p.w) {
        const Unit<P> w = param(p.w, e);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          g[j] += r * (dh.get(j) * w.get(j)) - back * x.get(j);
          nw[j] = dh.get(j) * (x.get(j) * r);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          g[j] += r * dh.get(j) - back * x.get(j);
          nw[j] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kUnit; j += 2) o.set2(j, g[j], g[j + 1]);
      if (p.dx) rowvec::store_unit<T>(static_cast<T*>(p.dx) + r0 * p.lddx + e, o, cols - e);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) np[j] = ng[j] = 0.f;
      if (p.y) {
        const Unit<T> y = load(p.y, p.ldy, e);
        const Unit<float> k = factor(e);
        if (p.wp) {
          const Unit<P> wp = param(p.wp, e);
#pragma unroll
          for (int j = 0; j < kUnit; j += 2) {
            float d[2];
#pragma unroll
            for (int l = 0; l < 2; ++l) {
              const float yn = y.get(j + l) * q, dz = g[j + l] * k.get(j + l);
              np[j + l] = dz * yn;
              ng[j + l] = g[j + l] * (yn * wp.get(j + l)) * p.scale;
              d[l] = q * (dz * wp.get(j + l)) - back2 * y.get(j + l);
            }
            o.set2(j, d[0], d[1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kUnit; j += 2) {
            ng[j] = g[j] * y.get(j) * p.scale;
            ng[j + 1] = g[j + 1] * y.get(j + 1) * p.scale;
            o.set2(j, g[j] * k.get(j), g[j + 1] * k.get(j + 1));
          }
        }
        if (p.dy) rowvec::store_unit<T>(static_cast<T*>(p.dy) + r0 * p.lddy + e, o, cols - e);
        if (p.dgate) {
#pragma unroll
          for (int j = 0; j < kUnit; j += 2) o.set2(j, ng[j], ng[j + 1]);
          rowvec::store_unit<T>(static_cast<T*>(p.dgate) + r0 * p.lddg + e, o, cols - e);
        }
      }
      // (Elements beyond the row are zeros; a row that is not there has no part, whatever its statistics.)
      if (live && e < p.cols) {
        if constexpr (HELD) {
#pragma unroll
          for (int j = 0; j < kUnit; ++j) {
            held[e + j] += nw[j];
            held[width + e + j] += np[j];
            held[2 * width + e + j] += ng[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < kUnit; ++j) { cw[j] += nw[j]; cp[j] += np[j]; cg[j] += ng[j]; }
        }
      }
    }
  }
  // ---- this CTA's column sums
  float* const out = p.parts + (int64_t)blockIdx.x * 3 * p.cols;
  if constexpr (!HELD) {
    const int e = tx * kUnit;
    for (int t = 0; t < (int)blockDim.y; ++t) {
      if ((int)threadIdx.y == t && e < p.cols) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          held[e + j] = t ? held[e + j] + cw[j] : cw[j];
          held[width + e + j] = t ? held[width + e + j] + cp[j] : cp[j];
          held[2 * width + e + j] = t ? held[2 * width + e + j] + cg[j] : cg[j];
        }
      }
      __syncthreads();
    }
  } else {
    __syncthreads();
  }
  const int all = TX * (int)blockDim.y, me = (int)threadIdx.y * TX + tx;
#pragma unroll
  for (int v = 0; v < 3; ++v)
    for (int i = me; i < p.cols; i += all) out[v * p.cols + i] = held[v * width + i];
}

struct ColumnParams {
  const float* parts;
  float* out[3];
  int32_t ctas, cols;
};
// Sums of the CTAs' parts: 32 columns of one output per block, 8 slices of the parts.
__global__ void __launch_bounds__(256) residual_norm_columns_kernel(const __grid_constant__ ColumnParams p) {
  __shared__ float slice[8][33];
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
  float* const out = p.out[blockIdx.y];
  if (!out) return;
  const int c = (int)blockIdx.x * 32 + (int)threadIdx.x;
  float s = 0.f;
  if (c < p.cols) {
    const float* const at = p.parts + (int64_t)blockIdx.y * p.cols + c;
#pragma unroll 8
    for (int i = (int)threadIdx.y; i < p.ctas; i += 8) s += at[(int64_t)i * 3 * p.cols];
  }
  slice[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < p.cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += slice[i][threadIdx.x];
    out[c] = s;
  }
}

// Threads of a row, rows of a CTA and CTAs of the backward pass.
struct BackShape {
  int tx, ty, ctas, held_bytes;
  bool held;
};
BackShape back_shape(int64_t rows, int64_t cols) {
  BackShape s;
  const int units = (int)((cols + kUnit - 1) / kUnit);
  s.held = units > kMaxThreads;
  s.tx = s.held ? kMaxThreads : (units + 31) / 32 * 32;
  s.ty = s.tx >= 256 ? 1 : 256 / s.tx;
  if (s.ty > rows) s.ty = rows < 1 ? 1 : (int)rows;
  const int64_t groups = (rows + s.ty - 1) / s.ty, most = 148 * (s.tx > 256 || s.held ? 1 : 2);
  s.ctas = (int)(groups < most ? groups : most);
  s.held_bytes = 3 * units * kUnit * 4;
  return s;
}

template <typename T, typename P>
cudaError_t launch_backward(const BackParams& p, const BackShape& s, cudaStream_t st) {
  const auto fn = s.held ? residual_norm_backward_kernel<T, P, true> : residual_norm_backward_kernel<T, P, false>;
  // (Always the same limit: calls of other sizes may be between this line and the launch.)
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * kMaxCols * 4);
  if (e != cudaSuccess) return e;
  return launch_overlapped(fn, dim3((unsigned)s.ctas), dim3((unsigned)s.tx, (unsigned)s.ty), (size_t)s.held_bytes, 1, st, p);
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
  p.x = a->x; p.ldx = a->ldx; p.y = a->y; p.ldy = a->ldy; p.xo = a->x_out; p.ldo = a->ldo; p.h = a->h; p.ldh = a->ldh;
  p.w = a->weight; p.wp = a->post_weight; p.gate = a->gate; p.ldg = a->gate ? a->ldg : 0;
  p.rows = a->rows; p.cols = (int32_t)a->cols; p.scale = a->scale; p.eps = a->eps;
  p.values = static_cast<uint8_t*>(a->values); p.ldv = a->ldv; p.scales = static_cast<uint8_t*>(a->scales); p.row_scale = a->row_scale;
  p.tiles = a->block ? fp4op::scale_tiles(a->cols, a->block) : 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(a->block ? a->values : a->h);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const bool p32 = a->param_type == GEMM_TYPE_FP32;
  if (a->type == GEMM_TYPE_BF16)
    return status_of(p32 ? launch_forward<__nv_bfloat16, float>(p, a->block, st) : launch_forward<__nv_bfloat16, __nv_bfloat16>(p, a->block, st));
  if (a->type == GEMM_TYPE_FP16) return status_of(p32 ? launch_forward<__half, float>(p, a->block, st) : launch_forward<__half, __half>(p, a->block, st));
  return status_of(launch_forward<float, float>(p, a->block, st));
}

extern "C" int64_t gemm_sm100a_residual_norm_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1 || cols > kMaxCols || rows > INT32_MAX / 2) return -1;
  return rows == 0 ? 0 : (int64_t)back_shape(rows, cols).ctas * 3 * cols * 4;
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
  const Mat ins[5] = {{a->dh, a->lddh}, {a->dx_out, a->lddo}, {a->x_out, a->ldo}, {a->y, a->ldy}, {matrix ? a->gate : nullptr, a->ldg}};
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
  const BackShape s = back_shape(a->rows, a->cols);
  if (a->workspace_bytes < (int64_t)s.ctas * 3 * a->cols * 4) return GEMM_ERR_BAD_ARGS;
  BackParams p;
  memset(&p, 0, sizeof(p));
  p.dh = a->dh; p.lddh = a->lddh; p.dxo = a->dx_out; p.lddo = a->lddo; p.xo = a->x_out; p.ldo = a->ldo; p.y = a->y; p.ldy = a->ldy;
  p.w = a->weight; p.wp = a->post_weight; p.gate = a->gate; p.ldg = a->gate ? a->ldg : 0;
  p.dx = a->dx; p.lddx = a->lddx; p.dy = a->dy; p.lddy = a->lddy; p.dgate = matrix ? a->dgate : nullptr; p.lddg = a->lddg;
  p.parts = static_cast<float*>(a->workspace);
  p.rows = a->rows; p.cols = (int32_t)a->cols; p.scale = a->scale; p.eps = a->eps;
  PointerDeviceGuard guard(a->dx);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const bool p32 = a->param_type == GEMM_TYPE_FP32;
  cudaError_t err;
  if (a->type == GEMM_TYPE_BF16) err = p32 ? launch_backward<__nv_bfloat16, float>(p, s, st) : launch_backward<__nv_bfloat16, __nv_bfloat16>(p, s, st);
  else if (a->type == GEMM_TYPE_FP16) err = p32 ? launch_backward<__half, float>(p, s, st) : launch_backward<__half, __half>(p, s, st);
  else err = launch_backward<float, float>(p, s, st);
  if (err == cudaSuccess && any) {
    ColumnParams c;
    c.parts = p.parts;
    for (int i = 0; i < 3; ++i) c.out[i] = sums[i];
    c.ctas = s.ctas;
    c.cols = p.cols;
    err = launch_overlapped(residual_norm_columns_kernel, dim3((unsigned)((p.cols + 31) / 32), 3), dim3(32, 8), 0, 1, st, c);
  }
  return status_of(err);
}
