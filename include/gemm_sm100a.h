/*
 * gemm_sm100a.h -- C ABI of the B200 (sm_100a) dense GEMM mainloop library.
 *
 * The library replaces the CUTLASS SM100 GEMM that the reference benchmark
 * cutlass_gemm_mainloop/cutlass_gemm_bench.cu instantiates (GEMM types at
 * cutlass_gemm_bench.cu:101-156) and drives through
 * Gemm::can_implement / initialize / run (cutlass_gemm_bench.cu:206-239).
 * The math is the reference's:
 *
 *     D = alpha * (A . B^T) + beta * C      (the reference runs beta = 0 with no C source,
 *                                            cutlass_gemm_bench.cu:117-118,196-204; its
 *                                            LinearCombination epilogue also takes beta and C)
 *
 *   A  M x K, row-major   (K contiguous)      cutlass_gemm_bench.cu:103 LayoutA = RowMajor
 *   B  N x K, "K-major"   (K contiguous)      cutlass_gemm_bench.cu:104 LayoutB = ColumnMajor (K x N)
 *   D  M x N, column-major (M contiguous), bf16  cutlass_gemm_bench.cu:105 LayoutD = ColumnMajor
 *   accumulate in fp32                         cutlass_gemm_bench.cu:69 ElementAccumulator = float
 *
 * Element types: bf16 and fp8 e4m3 as in the reference (DTYPE_ID 0 and 1,
 * cutlass_gemm_bench.cu:57-66), plus NVFP4 (DTYPE_ID 2): packed e2m1 values
 * with one unsigned e4m3 scale per 16 consecutive K elements of each row.
 *
 * Ownership: the caller owns every buffer (A, B, scale factors, D and the
 * optional status word). The launcher allocates nothing and throws nothing;
 * its only global state is a once-initialised driver entry point and a
 * mutex-guarded record of the kernels whose shared-memory limit it has raised
 * on each device, so concurrent calls on different streams or devices are safe.
 */
#ifndef GEMM_SM100A_H
#define GEMM_SM100A_H

#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element type selector; the numeric values equal the reference's DTYPE_ID
 * (cutlass_gemm_bench.cu:57-66) with NVFP4 appended. */
enum {
  GEMM_DTYPE_BF16     = 0,
  GEMM_DTYPE_FP8_E4M3 = 1,
  GEMM_DTYPE_NVFP4    = 2
};

/* Return codes. */
enum {
  GEMM_OK               = 0,
  GEMM_ERR_CANNOT_IMPLEMENT = -1,  /* shape, alignment, knob or smem limit (Gemm::can_implement, cutlass_gemm_bench.cu:211-218) */
  GEMM_ERR_LAUNCH       = -2,      /* CUDA launch / driver error (Gemm::initialize / run failure, cutlass_gemm_bench.cu:220-224) */
  GEMM_ERR_TIMEOUT      = -3,      /* a device-side bounded wait ran out; read back from the status word */
  GEMM_ERR_BAD_ARGS     = -4       /* null pointer, struct-size mismatch */
};

/* Layout of D (and C): the reference's LayoutD is column-major
 * (cutlass_gemm_bench.cu:105); row-major is the other LinearCombination layout. */
enum {
  GEMM_LAYOUT_COL_MAJOR = 0,   /* M contiguous, element (i, j) at i + j * ld */
  GEMM_LAYOUT_ROW_MAJOR = 1    /* N contiguous, element (i, j) at i * ld + j */
};

/* Flags. */
enum {
  /* Fault injection for tests of the timeout path: the producer warp issues
   * no loads, so every consumer wait runs out after timeout_ms and the kernel
   * records GEMM_ERR_TIMEOUT in *status and returns.  Never used for timing. */
  GEMM_FLAG_INJECT_STALL = 1u << 0,
  /* Store D straight from registers instead of staging each chunk in shared
   * memory for a TMA store (the fallback when the staging buffers do not fit
   * next to the ring); for comparisons of the two epilogues. */
  GEMM_FLAG_DIRECT_EPILOGUE = 1u << 1
};

/*
 * GemmArgs: one GEMM problem plus the kernel knobs.
 *
 * Knob names and defaults follow the reference's compile-time macros
 * (cutlass_gemm_bench.cu:34-49: TILE_M=128, TILE_N=128, TILE_K=64,
 * STAGES=0 meaning "auto", DTYPE_ID=0); here they are runtime fields.
 * cta_group (1 or 2) selects 1-SM or 2-SM (CTA pair) MMAs; cluster_m is the
 * number of CTAs per cluster along M and must equal cta_group (no load uses
 * cluster multicast).
 *
 * Leading dimensions are in ELEMENTS (for NVFP4, elements are 4-bit; lda and
 * ldb must then be even).  All base pointers must be 16-byte aligned and
 * lda*elem_bytes, ldb*elem_bytes, ldd*2 multiples of 16 (the reference's
 * 128-bit AlignmentA/B/D, cutlass_gemm_bench.cu:110-112).
 *
 * NVFP4 scale factors (sfa for A, sfb for B) are unsigned e4m3 bytes in the
 * 128-row x 4-scale interleaved atom layout: for row r and scale column c
 * (c = k / 16) the byte offset is
 *     ((r / 128) * (K / 64) + c / 4) * 512 + (r % 32) * 16 + ((r % 128) / 32) * 4 + (c % 4)
 * NVFP4 needs m a multiple of the MMA M (128, or 256 for cta_group 2), n a
 * multiple of tile_n and k a multiple of tile_k; the scale buffers then hold
 * (m / 128) * (k / 64) and (n / 128) * (k / 64) atoms of 512 bytes.
 */
typedef struct GemmArgs {
  uint32_t struct_size;   /* sizeof(GemmArgs), guards ABI drift */
  int32_t  dtype;         /* GEMM_DTYPE_* */
  int64_t  m, n, k;
  const void* a;  int64_t lda;
  const void* b;  int64_t ldb;
  void*       d;  int64_t ldd;
  const void* sfa;        /* NVFP4 only */
  const void* sfb;        /* NVFP4 only */
  float    alpha;         /* D = alpha * acc; 1.0 in the reference */
  int32_t  tile_m;        /* per-MMA M: 64 or 128 (cta_group 1), 256 (cta_group 2); 0 = default */
  int32_t  tile_n;        /* cta_group 1: 16, 32, 64, 128, 192, 256; cta_group 2: 64, 128, 192, 256, 512;
                             NVFP4: 128 or 256; 0 = default (256) */
  int32_t  tile_k;        /* K per pipeline stage: one or two 32-byte MMA K steps (bf16 16/32, fp8 32/64),
                             or 1, 2 or 4 128-byte swizzle atoms (bf16 64/128/256, fp8 128/256/512,
                             NVFP4 256/512/1024); 0 = one atom */
  int32_t  stages;        /* shared-memory ring depth; 0 = auto (as many as fit) */
  int32_t  cta_group;     /* 1 or 2; 0 = default (1) */
  int32_t  cluster_m;     /* CTAs per cluster along M; 0 = cta_group */
  int32_t  max_ctas;      /* grid cap; 0 = one CTA per SM (persistent); 1 = single-CTA mainloop mode */
  int32_t  raster_group;  /* tile order for L2 reuse: G > 0 groups of G M-tiles (M fastest), G < 0 groups of -G N-tiles (N fastest); 0 = default */
  int32_t* status;        /* optional device int32: 0 on success, GEMM_ERR_TIMEOUT (and where) on a device wait timeout */
  uint32_t timeout_ms;    /* device wait budget; 0 = default (4000 ms) */
  uint32_t flags;         /* GEMM_FLAG_* */
  int32_t  l2_prefetch;   /* warm L2 this many k-blocks ahead of the shared-memory ring; 0 = default, < 0 = off */
  unsigned long long* clock_out; /* optional device [2]: every CTA adds the SM cycles and nanoseconds it
                                    spent in the launch (zero it first; cycles / ns = the launch's mean
                                    effective SM clock under power capping) */
  /* Epilogue (CUTLASS LinearCombination, cutlass_gemm_bench.cu:117-118,196-204):
   * D = alpha * scale_a * scale_b * (A . B^T) + beta * C, computed in fp32 and
   * rounded once to bf16.  C is bf16 with D's layout and leading dimension ldc
   * (16-byte aligned, ldc a multiple of 8), read only when beta != 0; C may be D. */
  float    beta;          /* 0 in the reference */
  const void* c;          /* bf16 C, or NULL when beta == 0 */
  int64_t  ldc;
  int32_t  d_layout;      /* GEMM_LAYOUT_*; 0 = column-major as in the reference */
  float    scale_a;       /* per-tensor dequantisation scale of A (fp8: "per-tensor fp32 scale"); 0 means 1.0 */
  float    scale_b;       /* per-tensor scale of B; 0 means 1.0 */
} GemmArgs;

/* What a launch would do; filled by gemm_sm100a_query. */
typedef struct GemmInfo {
  uint32_t struct_size;
  int32_t  tile_m, tile_n, tile_k, stages, cta_group, cluster_m;
  int32_t  max_stages;           /* stages that fit in 227 KiB of shared memory */
  int64_t  smem_bytes_per_stage; /* per CTA */
  int64_t  smem_bytes;           /* dynamic shared memory per CTA */
  int32_t  tmem_columns;         /* tensor-memory columns allocated per CTA */
  int32_t  grid_ctas;            /* CTAs launched */
  int64_t  num_tiles;            /* output tiles (per CTA pair for cta_group 2) */
  int32_t  num_sms;
  int32_t  can_implement;        /* 1 if gemm_sm100a_launch would accept the arguments */
  char     reason[128];          /* why not, when can_implement == 0 */
  int32_t  epilogue_staging_buffers; /* shared-memory staging buffers per epilogue group (TMA-store
                                        epilogue); 0 = D stored directly from registers */
} GemmInfo;

/*
 * Validate the arguments and resolve defaults / auto stages without
 * launching.  Replaces Gemm::can_implement + Gemm::get_workspace_size
 * (cutlass_gemm_bench.cu:208-218); the workspace is always zero bytes.
 * Returns GEMM_OK or GEMM_ERR_CANNOT_IMPLEMENT / GEMM_ERR_BAD_ARGS.
 */
int gemm_sm100a_query(const GemmArgs* args, GemmInfo* info);

/*
 * Enqueue D = alpha * A . B^T on `stream` (a cudaStream_t; 0 = legacy default
 * stream).  Replaces Gemm::initialize + Gemm::run (cutlass_gemm_bench.cu:220-239):
 * each call encodes the TMA descriptors on the host and issues exactly one
 * kernel launch.  Asynchronous: a device wait timeout is reported through
 * args->status, read it with gemm_sm100a_read_status after synchronising.
 * Returns GEMM_OK, GEMM_ERR_CANNOT_IMPLEMENT, GEMM_ERR_BAD_ARGS or GEMM_ERR_LAUNCH.
 */
int gemm_sm100a_launch(const GemmArgs* args, void* stream);

/*
 * gemm_sm100a_launch, fused with an all-gather of D across the GPUs of one
 * box: the epilogue also stores every element of this launch's D block into
 * each of `n_peers` (at most 7) further buffers, typically the same block of
 * the full D on the other GPUs of an N-split, so the gather overlaps the GEMM
 * instead of following it (replaces the GEMM + ncclAllGather pair the N-split
 * harness otherwise issues; the reference is single-GPU and has none).
 * Each peer buffer uses args->ldd and must hold the same m x n block as
 * args->d (checked against its allocation before the launch); D must be
 * column-major (GEMM_ERR_CANNOT_IMPLEMENT otherwise).  Peer pointers must be device memory this GPU can reach: the call
 * enables peer access to other GPUs' memory and returns GEMM_ERR_BAD_ARGS for
 * host memory, unreachable devices or misaligned pointers.  Only D is
 * gathered; completion on every GPU means the full D is complete there.
 * It pays off while the D bytes each GPU sends are small next to its GEMM
 * time: on B200, config 5 split over 2 GPUs ran 33 % faster than GEMM +
 * ncclAllGather, over 8 GPUs 23 % slower (the epilogue's 64-byte stores move
 * ~370 GB/s per GPU over NVLink, NCCL ~580 GB/s).
 */
int gemm_sm100a_launch_gather(const GemmArgs* args, void* const* peer_d, int32_t n_peers, void* stream);

/*
 * Synchronise `stream`, copy the device status word back and map it to a
 * return code (GEMM_OK or GEMM_ERR_TIMEOUT); *detail (optional) receives the
 * raw word, which encodes the waiting role and pipeline stage.
 */
int gemm_sm100a_read_status(const int32_t* status, void* stream, int32_t* detail);

/* Static description of a return code. */
const char* gemm_sm100a_strerror(int code);

/* Library version, major*10000 + minor*100 + patch. */
int gemm_sm100a_version(void);

/*
 * Seeded input generation on the device (harness helper, not part of the
 * GEMM).  Every element is a pure function of (seed, stream_id, index), so
 * any GPU can regenerate any slice of a matrix and a host checker can
 * regenerate any element.
 *   dist: 0 = uniform[-1,1), 1 = normal(0,1)
 *   out_dtype: GEMM_DTYPE_BF16 or GEMM_DTYPE_FP8_E4M3 (round to nearest even,
 *   fp8 saturating); values are multiplied by `scale` before rounding.
 * Generates rows [row0, row0+rows) of a rows_total x cols row-major matrix
 * (row stride ld elements); element (r, c) uses index r*cols + c.
 */
int gemm_sm100a_generate(void* out, int32_t out_dtype, int32_t dist, float scale,
                         uint64_t seed, uint64_t stream_id,
                         int64_t row0, int64_t rows, int64_t cols, int64_t ld,
                         void* cuda_stream);

/*
 * NVFP4 quantisation of a seeded normal(0,1)*scale matrix on the device:
 * writes packed e2m1 values (two per byte, low nibble = even column) and the
 * unsigned-e4m3 block scales (absmax/6 rounded up) in the interleaved layout
 * described above.  Rows [row0, row0+rows) of a matrix with `cols` columns
 * (cols a multiple of 64, row0 and rows multiples of 128).
 */
int gemm_sm100a_generate_nvfp4(void* out_packed, void* out_scales, float scale,
                               uint64_t seed, uint64_t stream_id,
                               int64_t row0, int64_t rows, int64_t cols,
                               void* cuda_stream);

/*
 * Measured tcgen05 dense peak (replaces the reference's umma_throughput/umma_tput.cu
 * probe, kernel :286-544, with an NVFP4 kind and a whole-GPU mode added).
 * Launches `num_ctas` CTAs (a multiple of cta_group; one per SM at most), each
 * issuing `iters` groups of `depth` back-to-back M=128*cta_group, N=256 MMAs of
 * `dtype` from shared memory, one commit per group.  results (device, caller-owned,
 * 3*num_ctas uint64) receives per CTA {clock64 cycles, %globaltimer ns, status}
 * (zeros for the non-issuing CTA of a pair).  Returns GEMM_OK, GEMM_ERR_BAD_ARGS
 * or GEMM_ERR_LAUNCH; asynchronous on `stream`.
 */
int gemm_sm100a_umma_peak(int32_t dtype, int32_t cta_group, int32_t num_ctas, int32_t depth,
                          int32_t iters, unsigned long long* results, void* stream);

/*
 * TMA-2D HBM read-throughput probe (replaces the reference's
 * tma2d_throughput/tma2d_tput.cu: kernel :42-126, launch :131-219).  Launches
 * ctas_per_sm one-warp CTAs per SM (227 KiB of shared memory each, as the
 * reference pins it), which stream the 32-bit words of `buf` (read as a
 * (bytes / (4 * box_width)) x box_width row-major tensor, whole box_rows-row
 * tiles only) through a `stages`-deep ring of (box_rows x box_width) TMA
 * tiles.  results (device, caller-owned, 5 * num_SMs * ctas_per_sm uint64)
 * receives per CTA {clock64 cycles, %globaltimer ns, tiles loaded, XOR of the
 * first 32 words of every tile it loaded, status (0, or 3 if a load wait ran
 * out after 2 s)}.  box_width: 4..256 words, a multiple of 4; box_rows 1..256;
 * tiles of at least 128 bytes.  Time it with events on `stream` after
 * flushing L2: bytes / time is the TMA read roof.  Returns GEMM_OK,
 * GEMM_ERR_BAD_ARGS, GEMM_ERR_CANNOT_IMPLEMENT (ring over shared memory) or
 * GEMM_ERR_LAUNCH; asynchronous.
 */
int gemm_sm100a_tma_read_probe(const void* buf, int64_t bytes, int32_t box_width, int32_t box_rows,
                               int32_t stages, int32_t ctas_per_sm, unsigned long long* results, void* stream);

/* ------------------------------------------------------------------------
 * 8-bit integer linear layers: the product of int8 operands with one scale per
 * token and channel, the quantiser that makes such operands, and dropout.
 * ------------------------------------------------------------------------ */

/* Element types of the floating tensors these calls read and write. */
enum {
  GEMM_TYPE_BF16 = 0,
  GEMM_TYPE_FP16 = 1,
  GEMM_TYPE_FP32 = 2
};

/*
 * Dropout of element (r, c) of a matrix, from the generator's counter (see
 * gemm_sm100a_generate): nothing is stored, the mask is a pure function of
 * (seed, stream_id, index), so the backward pass and every rank of an N-split
 * regenerate exactly their part of it.
 *   index = (row0 + r) * row_elems + col0 + c
 *   h     = mix64(key(seed, stream_id) + (index / 2 + 1) * 0x9E3779B97F4A7C15)
 *   word  = index odd ? h >> 32 : h & 0xFFFFFFFF
 *   kept iff word >= rint(p * 2^32); a kept value is multiplied by 1 / (1 - p),
 *   a dropped one is replaced by 0 whatever it was (NaN and Inf included).
 * p = 0 disables it (no other field is read), p = 1 drops everything.
 * row0, col0 >= 0, row_elems >= col0 + columns, all indices below 2^62.
 */
typedef struct DropoutArgs {
  double   p;
  uint64_t seed, stream_id;
  const uint64_t* seed_offset; /* optional device word added to seed when the kernel runs, so that
                                  a captured graph draws a new mask at each replay; 8-byte aligned */
  int64_t  row0, col0, row_elems;
} DropoutArgs;

/*
 *   D = C + dropout( scale_a[i] * scale_b[j] * sum_k A[i][k] B[j][k] + bias[j] )
 *
 *   A  m x k int8 (tokens), B  n x k int8 (channels), K contiguous, rows of
 *   lda / ldb bytes (multiples of 16, bases 16-byte aligned); bytes between k
 *   and the row stride are not used.  The sum is exact in int32 (k <= 131071),
 *   everything after it fp32, rounded once to d_type (scale_b first where
 *   |scale_a| > 2^96, which alone could take the sum out of range).  The result has the
 *   same bits for every tile, split and size of the batch.
 *   scale_a (m) and scale_b (n) fp32; NULL means 1.
 *   D  m x n row-major (N contiguous), leading dimension ldd >= n elements,
 *   any alignment of its own type; C (optional) like D with ldc, is D (same
 *   stride) or does not overlap it (else refused).
 *   bias (optional): n elements of bias_type.
 * m or n of 0: nothing is launched.  D must not overlap A, B, scales or bias.
 */
typedef struct Int8GemmArgs {
  uint32_t struct_size;    /* sizeof(Int8GemmArgs) */
  int32_t  d_type;         /* GEMM_TYPE_*: D and C */
  int64_t  m, n, k;
  const void* a;  int64_t lda;
  const void* b;  int64_t ldb;
  void*       d;  int64_t ldd;
  const void* c;  int64_t ldc;
  const float* scale_a;
  const float* scale_b;
  const void* bias;
  int32_t  bias_type;      /* GEMM_TYPE_* */
  int32_t  tile_n;         /* tokens per tile; 0 = chosen from the sizes */
  int32_t  cta_group;      /* 1 or 2 (CTA pair); 0 = chosen */
  int32_t  split_k;        /* CTAs that share one tile's K; 0 = chosen */
  DropoutArgs drop;
  int32_t* status;         /* optional device int32, as in GemmArgs */
  uint32_t timeout_ms;     /* device wait budget; 0 = 4000 ms */
  uint32_t flags;          /* 0 or GEMM_FLAG_INJECT_STALL */
} Int8GemmArgs;

/* Validate and resolve gemm_sm100a_int8_launch without launching (GemmInfo.tile_m is the
 * channels of a tile, tile_n its tokens).  The one-launch form of the linear layer below has
 * its own tiles and is not described. */
int gemm_sm100a_int8_query(const Int8GemmArgs* args, GemmInfo* info);

/* Enqueue one product; asynchronous, allocates nothing, capturable. */
int gemm_sm100a_int8_launch(const Int8GemmArgs* args, void* stream);

/*
 * Quantise the rows of X (m x k of x_type, row stride ldx elements) and multiply:
 * gemm_sm100a_quantize_int8 followed by gemm_sm100a_int8_launch, bit for bit, in one
 * or two launches.  args->a and args->scale_a are workspace of the caller
 * (m * lda bytes and m floats; their content afterwards is unspecified).  They
 * may be NULL where one launch quantises and multiplies: x_type equal to d_type,
 * m <= 8, m * k <= 16384, no knob or flag set and D apart from X.
 * D may lie over X, with X as C too (the layer's result replaces its tokens).
 */
int gemm_sm100a_int8_linear(const Int8GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream);

/*
 * Symmetric int8 quantisation with one scale per row:
 *   amax_i = max(max_j |x_ij|, 127 * 2^-126),  scale_i = amax_i / 127,
 *   q_ij   = 127 * x_ij / amax_i rounded to the nearest integer, ties to even
 * (decided exactly, not from a rounded quotient).  A row with a NaN or an
 * infinity gets that as its scale and zeros as q, which makes NaN of what is
 * computed from it and touches no other row.
 * With transpose: one scale per COLUMN, q stored cols x rows (ldq >= rows), and
 * optionally the sum of each column (fp32) in col_sums.
 * With drop.p > 0, x is first masked; the factor 1 / (1 - p) enters scale and
 * col_sums (indices count elements of X as stored, transposed or not).
 * q, scale and col_sums overlap neither X nor one another.
 * ldq is a multiple of 16 bytes, q 16-byte aligned; bytes of q beyond the last
 * element of a row are left as they were.  rows or cols of 0: with transpose
 * and rows = 0 the scales are 2^-126 and the sums 0, else nothing is written.
 */
typedef struct Int8QuantArgs {
  uint32_t struct_size;    /* sizeof(Int8QuantArgs) */
  int32_t  x_type;         /* GEMM_TYPE_* */
  int64_t  rows, cols;
  const void* x;  int64_t ldx;
  void*    q;     int64_t ldq;
  float*   scale;
  float*   col_sums;       /* transpose only; NULL = not wanted */
  int32_t  transpose;
  int32_t  reserved;       /* 0 */
  DropoutArgs drop;
} Int8QuantArgs;

int gemm_sm100a_quantize_int8(const Int8QuantArgs* args, void* stream);

/*
 * Gradients of y = residual + dropout(x . w^T + bias) for dY, by int8 products (the
 * straight-through gradient of the quantised layer):
 *   dZ = dropout(dY), dX = dZ . W, dW = dZ^T . X, dbias = column sums of dZ (fp32)
 * dY m x n, X and dX m x k of `type`; wt k x n int8 and wt_scale (k): W quantised
 * with transpose = 1; dW n x k of dw_type.  dx, dw and dbias may each be NULL (not
 * wanted; wt is read for dx only, x for dw only).  m, n <= 131071 (sums over them).
 * workspace: gemm_sm100a_int8_backward_workspace(m, n, k) bytes, 16-byte aligned,
 * of this call alone until it has run.  dX and dW may lie over X or dY, not over each
 * other, wt or wt_scale; dbias and the workspace overlap nothing.  m = 0 sets dW and dbias to 0.
 * Refusals come before the first launch.  Asynchronous, capturable.
 */
typedef struct Int8BackwardArgs {
  uint32_t struct_size;    /* sizeof(Int8BackwardArgs) */
  int32_t  type;           /* GEMM_TYPE_*: dY, X and dX */
  int64_t  m, n, k;
  const void* dy;  int64_t lddy;
  const void* x;   int64_t ldx;
  const void* wt;  int64_t ldwt;
  const float* wt_scale;
  void*    dx;     int64_t lddx;
  void*    dw;     int64_t lddw;
  float*   dbias;
  int32_t  dw_type;        /* GEMM_TYPE_* */
  int32_t  reserved;       /* 0 */
  void*    workspace;  int64_t workspace_bytes;
  DropoutArgs drop;
  int32_t* status;         /* optional, as in Int8GemmArgs */
} Int8BackwardArgs;

/* Bytes of workspace, -1 for sizes that are refused. */
int64_t gemm_sm100a_int8_backward_workspace(int64_t m, int64_t n, int64_t k);

int gemm_sm100a_int8_linear_backward(const Int8BackwardArgs* args, void* stream);

/*
 * Y = residual + dropout(X), rows x cols row-major with their own row strides
 * (elements), all of one type, any alignment of that type; computed in fp32 and
 * rounded once.  Its gradient is the same call on dY without the residual.
 * Y may be X or residual (same stride); Y that overlaps one of them in another way
 * is refused.
 */
typedef struct DropoutOpArgs {
  uint32_t struct_size;    /* sizeof(DropoutOpArgs) */
  int32_t  type;           /* GEMM_TYPE_* */
  int64_t  rows, cols;
  const void* x;         int64_t ldx;
  const void* residual;  int64_t ldr;   /* NULL = none */
  void*    y;            int64_t ldy;
  DropoutArgs drop;
} DropoutOpArgs;

int gemm_sm100a_dropout(const DropoutOpArgs* args, void* stream);

/* ------------------------------------------------------------------------
 * 4-bit floating linear layers: e2m1 values with a scale for each block of 16
 * or 32 elements along K and one for each row, their quantiser and product.
 * ------------------------------------------------------------------------ */

/*
 * A 4-bit matrix of rows x cols:
 *   values     two to a byte, the even column in the low four bits; row stride in bytes.  With an odd
 *              number of columns the last byte's high bits are 0.
 *   scales     block 16: unsigned e4m3, block 32: e8m0 (2^(byte - 127)).  In tiles of 128 rows x 4
 *              scales: row r, block column c at byte
 *                ((r / 128) * tiles + c / 4) * 512 + (r % 32) * 16 + ((r % 128) / 32) * 4 + c % 4
 *              with tiles = ceil(cols / 256) * (block == 16 ? 4 : 2), 16-byte aligned.  The scales of the
 *              block columns beyond cols are stored too and must not be NaN (the quantiser writes
 *              0, or 1 for e8m0); those of rows beyond the last are not used.
 *              (For columns in multiples of 256 this is the layout of GemmArgs.sfa.)
 *   row_scale  fp32, one for each row.
 * An element stands for value * scale * row_scale.
 */

/* Bytes of the scales of a rows x cols matrix, -1 for sizes that are refused. */
int64_t gemm_sm100a_fp4_scale_bytes(int64_t rows, int64_t cols, int32_t block);

/*
 * Quantise the rows of X:
 *   row_scale g = 2^(floor(log2 max|x|) - 10), at least 2^-126;  y = x / g in fp32 (exact from 2^-126 on)
 *   scale     s = the least e4m3 number (block 16) or power of two from 2^-126 on (block 32) with
 *                 6 s >= max|y| over the block (so nothing is clipped; the OCP conversion to blocks of 32 takes
 *                 2^(floor(log2 max) - 2) and saturates)
 *   value     q = y / s rounded to e2m1, ties to the even code, decided exactly
 * A row with a NaN or an infinity gets that as its row scale and zeros as values: what is computed from
 * it is NaN, and no other row is touched.  The three outputs overlap neither X nor one another.
 * values is 16-byte aligned, ldv a multiple of 16; bytes behind a row's last element are left as they were.
 */
typedef struct Fp4QuantArgs {
  uint32_t struct_size;    /* sizeof(Fp4QuantArgs) */
  int32_t  x_type;         /* GEMM_TYPE_* */
  int64_t  rows, cols;
  const void* x;       int64_t ldx;
  void*    values;     int64_t ldv;   /* bytes */
  void*    scales;
  float*   row_scale;
  int32_t  block;          /* 16 or 32 */
  int32_t  reserved;       /* 0 */
} Fp4QuantArgs;

int gemm_sm100a_quantize_fp4(const Fp4QuantArgs* args, void* stream);

/* Y = value * scale * row_scale (row_scale NULL: 1), computed in fp32, where powers of two as row scales keep it
 * exact unless it leaves fp32's range, and rounded to y_type. */
typedef struct Fp4DequantArgs {
  uint32_t struct_size;    /* sizeof(Fp4DequantArgs) */
  int32_t  y_type;         /* GEMM_TYPE_* */
  int64_t  rows, cols;
  const void* values;  int64_t ldv;   /* bytes */
  const void* scales;
  const float* row_scale;
  void*    y;          int64_t ldy;
  int32_t  block;
  int32_t  reserved;       /* 0 */
} Fp4DequantArgs;

int gemm_sm100a_dequantize_fp4(const Fp4DequantArgs* args, void* stream);

/*
 *   D = C + a_row_scale[i] * b_row_scale[j] * sum_k A[i][k] B[j][k] + bias[j]
 *
 * A  m x k (tokens) and B  n x k (channels), 4-bit, with one block size; values 16-byte aligned,
 * lda / ldb in bytes and multiples of 16 (bytes behind the last element's are not used).  Products and
 * block scales are exact; the sum is the tensor cores' fp32, whose order depends on the tile and the
 * split; the row scales, bias and residual fp32, rounded once to d_type (bf16 or fp16: fp32's last
 * bits are not in the sum).  Row scales NULL: 1.
 * D and C as in Int8GemmArgs: m x n row-major, any alignment of their type, C is D or lies apart from it.
 * m or n of 0: nothing is launched.  D must not overlap any other operand.
 */
typedef struct Fp4GemmArgs {
  uint32_t struct_size;    /* sizeof(Fp4GemmArgs) */
  int32_t  d_type;         /* GEMM_TYPE_BF16 or GEMM_TYPE_FP16: D and C */
  int64_t  m, n, k;
  const void* a;  int64_t lda;
  const void* a_scales;
  const float* a_row_scale;
  const void* b;  int64_t ldb;
  const void* b_scales;
  const float* b_row_scale;
  void*       d;  int64_t ldd;
  const void* c;  int64_t ldc;
  const void* bias;
  int32_t  bias_type;      /* GEMM_TYPE_* */
  int32_t  block;          /* 16 or 32 */
  int32_t  tile_n;         /* tokens per tile; 0 = chosen from the sizes */
  int32_t  cta_group;      /* 1 or 2 (CTA pair); 0 = chosen */
  int32_t  split_k;        /* CTAs that share one tile's K; 0 = chosen */
  int32_t  reserved;       /* 0 */
  int32_t* status;         /* optional device int32, as in GemmArgs */
  uint32_t timeout_ms;     /* device wait budget; 0 = 4000 ms */
  uint32_t flags;          /* 0 or GEMM_FLAG_INJECT_STALL */
} Fp4GemmArgs;

/* Validate and resolve gemm_sm100a_fp4_launch without launching (GemmInfo.tile_m is the channels of a
 * tile, tile_n its tokens). */
int gemm_sm100a_fp4_query(const Fp4GemmArgs* args, GemmInfo* info);

/* Enqueue one product; asynchronous, allocates nothing, capturable. */
int gemm_sm100a_fp4_launch(const Fp4GemmArgs* args, void* stream);

/*
 * Quantise the rows of X (m x k of x_type, row stride ldx elements) and multiply, in one or two launches.
 * args->a, a_scales and a_row_scale are workspace of the caller (m * lda bytes,
 * gemm_sm100a_fp4_scale_bytes(m, k, block) bytes, m floats; their content afterwards is unspecified).
 * They may be NULL where one launch quantises and multiplies: gemm_sm100a_fp4_linear_workspace == 0.
 * D may lie over X, with X as C too.
 */
int gemm_sm100a_fp4_linear(const Fp4GemmArgs* args, const void* x, int32_t x_type, int64_t ldx, void* stream);

/* Whether gemm_sm100a_fp4_linear reads args->a, a_scales and a_row_scale (1) or needs no workspace (0). */
int gemm_sm100a_fp4_linear_workspace(const Fp4GemmArgs* args, const void* x, int32_t x_type, int64_t ldx);

/* ------------------------------------------------------------------------
 * The residual stream around a block: the norm after it, its gate and scale, the
 * stream's update and the norm before the next block.
 * ------------------------------------------------------------------------ */

/*
 *   z     = post_weight ? y * r(y) * post_weight : y
 *   x_out = x + (gate * scale) * z                          rounded to `type`
 *   h     = x_out * r(x_out) * weight                       of the rounded x_out
 *   r(v)  = 1 / sqrt(mean(v^2) + eps) of a row
 * One fp32 operation after the other, from left to right; the mean in 64 bits (2^-40 or better of its value).
 * x, y, x_out, h and a gate matrix are of `type`, rows x cols with their own strides (elements), any alignment of
 * that type; weight, post_weight and a gate vector (ldg = 0) have cols elements of param_type: `type` or fp32.
 * weight NULL: 1.  gate NULL: 1.  y NULL: x_out is x, which is not written again (x_out NULL too).
 * block 16 or 32: h, before any rounding, becomes a 4-bit matrix (values, scales, row_scale as in Fp4QuantArgs; h is NULL).
 * cols <= 16384.  x_out may be x or y (same stride); otherwise outputs overlap nothing.
 */
typedef struct ResidualNormArgs {
  uint32_t struct_size;    /* sizeof(ResidualNormArgs) */
  int32_t  type;           /* GEMM_TYPE_* */
  int64_t  rows, cols;
  const void* x;       int64_t ldx;
  const void* y;       int64_t ldy;
  void*    x_out;      int64_t ldo;
  void*    h;          int64_t ldh;
  const void* weight;
  const void* post_weight;
  const void* gate;    int64_t ldg;   /* 0: a vector */
  int32_t  param_type;
  int32_t  block;          /* 0: h is floating */
  double   eps;            /* >= 0 */
  float    scale;
  int32_t  reserved;       /* 0 */
  void*    values;     int64_t ldv;
  void*    scales;
  float*   row_scale;
} ResidualNormArgs;

int gemm_sm100a_residual_norm(const ResidualNormArgs* args, void* stream);

/*
 * Its gradients, for dh and dx_out (NULL: 0) and the x_out, y, weights, gate, scale and eps of the call:
 *   g    = dx_out + the gradient of h towards x_out        dx = g
 *   dy   = the gradient of (gate * scale) * z towards y for g
 * of `type`, and the fp32 sums over rows dweight, dpost_weight and, for a gate vector, dgate; a gate
 * matrix has dgate of `type` (lddg).  y NULL: no dy, dpost_weight, dgate.  dweight, dpost_weight and dgate may be NULL
 * (not wanted).  The same call takes its sums in the same order.  rows = 0 sets the fp32 sums to 0.
 * Sums over a row or over rows are fp32, of fp32 rows too (a few 2^-24 of what they add up); those of a row far from one, whose
 * squares sum to 1e20 or more (or, with an eps below 1e-12, to 1e-20 or less) or whose products leave fp32's range, are 64-bit.
 * workspace: gemm_sm100a_residual_norm_workspace(rows, cols) bytes, 16-byte aligned, of this call alone until it has
 * run.  Outputs overlap nothing.
 */
typedef struct ResidualNormBackwardArgs {
  uint32_t struct_size;    /* sizeof(ResidualNormBackwardArgs) */
  int32_t  type;
  int64_t  rows, cols;
  const void* dh;      int64_t lddh;
  const void* dx_out;  int64_t lddo;
  const void* x_out;   int64_t ldo;
  const void* y;       int64_t ldy;
  const void* weight;
  const void* post_weight;
  const void* gate;    int64_t ldg;   /* 0: a vector */
  int32_t  param_type;
  float    scale;
  double   eps;
  void*    dx;         int64_t lddx;
  void*    dy;         int64_t lddy;
  float*   dweight;
  float*   dpost_weight;
  void*    dgate;      int64_t lddg;
  void*    workspace;  int64_t workspace_bytes;
} ResidualNormBackwardArgs;

/* Bytes of workspace, -1 for sizes that are refused. */
int64_t gemm_sm100a_residual_norm_workspace(int64_t rows, int64_t cols);

int gemm_sm100a_residual_norm_backward(const ResidualNormBackwardArgs* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GEMM_SM100A_H */
