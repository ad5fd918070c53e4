// int8_gemm.cu -- product of int8 operands with one scale per token and channel:
//   D[i][j] = C[i][j] + dropout(sa[i] * sb[j] * sum_k A[i][k] B[j][k] + bias[j])
// The sum is exact in int32, so every tiling gives the same bits.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>

#include "device_guard.cuh"
#include "gemm_sm100a.h"
#include "int8_common.cuh"

using namespace int8op;

namespace {

struct Int8Params {
  const int8_t* a; int64_t lda;
  const int8_t* b; int64_t ldb;
  void* d; int64_t ldd;
  const void* c; int64_t ldc;
  const float* sa;
  const float* sb;
  const void* bias;
  int32_t bias_type;
  int32_t m, n, k;
  Drop drop;
};

// One output from its exact sum.
__device__ __forceinline__ float finish(const Int8Params& p, int32_t acc, float sa, float sb, float bias, bool kept) {
  const float v = fmaf(__int2float_rn(acc) * sa, sb, bias);
  return !p.drop.on ? v : (kept ? v * p.drop.grow : 0.f);
}

// One thread per output, four products per instruction.
template <typename T>
__global__ void __launch_bounds__(256) int8_gemm_simple(const __grid_constant__ Int8Params p) {
  const int64_t j = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int64_t i = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5);
  if (i >= p.m || j >= p.n) return;
  const int8_t* a = p.a + i * p.lda;
  const int8_t* b = p.b + j * p.ldb;
  int32_t acc = 0;
  int k = 0;
  for (; k + 16 <= p.k; k += 16) {
    const int4 x = *reinterpret_cast<const int4*>(a + k), y = *reinterpret_cast<const int4*>(b + k);
    acc = __dp4a(x.x, y.x, __dp4a(x.y, y.y, __dp4a(x.z, y.z, __dp4a(x.w, y.w, acc))));
  }
  for (; k < p.k; ++k) acc += (int32_t)a[k] * b[k];
  const bool kept = !p.drop.on || drop_keeps(drop_key(p.drop), p.drop.threshold, drop_index(p.drop, i, j));
  float v = finish(p, acc, p.sa ? p.sa[i] : 1.f, p.sb ? p.sb[j] : 1.f, p.bias ? load_as_f32(p.bias, p.bias_type, j) : 0.f, kept);
  if (p.c) v += to_f32(static_cast<const T*>(p.c)[i * p.ldc + j]);
  static_cast<T*>(p.d)[i * p.ldd + j] = from_f32<T>(v);
}

struct Resolved {
  Int8Params p;
  char reason[128];
};

#define FAIL(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_CANNOT_IMPLEMENT; } while (0)
#define BAD(...) do { snprintf(r.reason, sizeof(r.reason), __VA_ARGS__); return GEMM_ERR_BAD_ARGS; } while (0)

int resolve(const Int8GemmArgs* a, Resolved& r) {
  memset(&r, 0, sizeof(r));
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
    if (!a->a || !a->b || !a->d) BAD("null A/B/D pointer");
    if ((reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->b)) & 15) FAIL("A/B must be 16-byte aligned");
    if (a->lda < a->k || a->ldb < a->k) FAIL("lda/ldb must be >= k");
    if ((a->lda | a->ldb) & 15) FAIL("lda/ldb must be multiples of 16");
    const uintptr_t e = (uintptr_t)type_bytes(a->d_type);
    if ((reinterpret_cast<uintptr_t>(a->d) | reinterpret_cast<uintptr_t>(a->c)) % e) FAIL("D/C must be aligned to their element");
    if (a->ldd < a->n) FAIL("ldd must be >= n");
    if (a->c && a->ldc < a->n) FAIL("ldc must be >= n");
    if ((reinterpret_cast<uintptr_t>(a->scale_a) | reinterpret_cast<uintptr_t>(a->scale_b)) & 3) FAIL("scales must be 4-byte aligned");
    if (a->bias && reinterpret_cast<uintptr_t>(a->bias) % type_bytes(a->bias_type)) FAIL("bias must be aligned to its element");
  }
  Int8Params& p = r.p;
  p.a = static_cast<const int8_t*>(a->a); p.lda = a->lda;
  p.b = static_cast<const int8_t*>(a->b); p.ldb = a->ldb;
  p.d = a->d; p.ldd = a->ldd; p.c = a->c; p.ldc = a->ldc;
  p.sa = a->scale_a; p.sb = a->scale_b; p.bias = a->bias; p.bias_type = a->bias_type;
  p.m = (int32_t)a->m; p.n = (int32_t)a->n; p.k = (int32_t)a->k;
  return GEMM_OK;
}

}  // namespace

extern "C" int gemm_sm100a_int8_query(const Int8GemmArgs* args, GemmInfo* info) {
  Resolved r;
  const int rc = resolve(args, r);
  if (info) {
    memset(info, 0, sizeof(*info));
    info->struct_size = sizeof(GemmInfo);
    info->can_implement = rc == GEMM_OK;
    memcpy(info->reason, r.reason, sizeof(info->reason));
  }
  return rc;
}

extern "C" int gemm_sm100a_int8_launch(const Int8GemmArgs* args, void* stream) {
  Resolved r;
  const int rc = resolve(args, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PointerDeviceGuard guard(args->d);
  if (!guard.ok) return GEMM_ERR_LAUNCH;
  const dim3 grid((unsigned)((args->n + 31) / 32), (unsigned)((args->m + 7) / 8));
  if (args->d_type == GEMM_TYPE_BF16) int8_gemm_simple<__nv_bfloat16><<<grid, 256, 0, st>>>(r.p);
  else if (args->d_type == GEMM_TYPE_FP16) int8_gemm_simple<__half><<<grid, 256, 0, st>>>(r.p);
  else int8_gemm_simple<float><<<grid, 256, 0, st>>>(r.p);
  if (cudaGetLastError() != cudaSuccess) return GEMM_ERR_LAUNCH;
  return GEMM_OK;
}

extern "C" int gemm_sm100a_int8_linear(const Int8GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream) {
  Resolved r;
  const int rc = resolve(args, r);
  if (rc != GEMM_OK) return rc;
  if (args->m == 0 || args->n == 0) return GEMM_OK;
  Int8QuantArgs q;
  memset(&q, 0, sizeof(q));
  q.struct_size = sizeof(q);
  q.x_type = x_type; q.rows = args->m; q.cols = args->k; q.x = x; q.ldx = ldx;
  q.q = const_cast<void*>(args->a); q.ldq = args->lda; q.scale = const_cast<float*>(args->scale_a);
  const int rq = gemm_sm100a_quantize_int8(&q, stream);
  return rq != GEMM_OK ? rq : gemm_sm100a_int8_launch(args, stream);
}
