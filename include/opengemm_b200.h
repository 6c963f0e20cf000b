/* C ABI of libopengemm_b200.so: a B200 (sm_100a) GEMM library that stands in
 * for both of OpenGEMM's kernel libraries.
 *
 * It exports, with the same names, signatures and status codes, the twelve
 * entry points the reference's front end binds through ctypes
 * (opengemm/python/capi.py:86-174): six for the dense library
 * (opengemm/src/mm/capi.h:9-17, opengemm/src/mm/capi.cu:6-32) and six for the
 * block-scaled one (opengemm/src/smm/capi.h:9-17, opengemm/src/smm/capi.cu:6-32).
 * Pointing OPENGEMM_LIB_MM and OPENGEMM_LIB_SMM (opengemm/python/build.py:100-102)
 * at this one file makes the unmodified reference front end run on it.
 *
 * Plain C: pointers and sizes only.  All data pointers are device pointers
 * owned by the caller; the library keeps no reference to them after a call
 * returns.  It allocates no device memory, with one exception: the first launch
 * on a device that asks for the stream-K schedule (split_k >= 2) allocates
 * that schedule's scratch (about 76 MB) for the life of the process, unless
 * og_b200_prepare_device did so earlier.  Launches are asynchronous on the
 * stream given.  Devices 0..63 are served.
 */
#ifndef OPENGEMM_B200_H
#define OPENGEMM_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(_WIN32)
#define OG_API __declspec(dllexport)
#else
#define OG_API __attribute__((visibility("default")))
#endif

/* opengemm/src/common/abi.h:11 */
#define OG_ABI_VERSION 3

/* Status codes, opengemm/src/common/abi.h:13-19; OG_ERR_TIMEOUT is new. */
enum {
  OG_OK = 0,
  OG_ERR_BIND = -1,      /* unknown dtype, or a K the format cannot take */
  OG_ERR_NO_KERNEL = -2, /* no kernel can serve the configuration */
  OG_ERR_TENSORMAP = -3,
  OG_ERR_LAUNCH = -4,
  OG_ERR_TIMEOUT = -5    /* a device-side wait ran out: what og_b200_status answers for a non-zero status word */
};

/* One GEMM: shape, the configs.json entry that picks and drives the kernel,
 * and the row og_*_bind resolved.  Field for field the reference's struct
 * (opengemm/src/common/abi.h:24-39), 108 bytes, no padding.  The caller fills
 * every field but `row`. */
typedef struct {
  int32_t m, n, k; /* k in values, not bytes */
  char dtype[16];  /* "bf16", "e4m3xe5m2", "nvfp4", ... */

  int32_t use_2cta, output_n, use_clc, swap_ab;
  int32_t cluster_m, cluster_n, cluster_k;
  int32_t block_m, stages, epi_hold, epi_double, epi_direct;
  int32_t epi_trade, deep_stages;

  int32_t supergroup, split_k, walk, l2_promo;
  int32_t persistent;

  int32_t row; /* set by og_*_bind */
} OgGemm;

/* ---- dense library: replaces opengemm/src/mm/capi.cu:6-32 ---------------- */

/* ABI version this library speaks (mm/capi.cu:6). */
OG_API int32_t og_mm_abi(void);
/* Text of the last failure on the calling thread (mm/capi.cu:8). */
OG_API const char* og_mm_error(void);
/* Number of kernel rows og_mm_kernel enumerates (mm/capi.cu:10). */
OG_API int32_t og_mm_kernels(void);
/* Fill `out` with the configuration that binds to row `i` (mm/capi.cu:12-18). */
OG_API int32_t og_mm_kernel(int32_t i, OgGemm* out);
/* Validate dtype / shape / knobs, clamp split_k, set g->row (mm/capi.cu:20, mm/launch.cuh:41-64). */
OG_API int32_t og_mm_bind(OgGemm* g);
/* Enqueue C[m,n] = A[m,k] . B[n,k]^T on `stream` of `device` (mm/capi.cu:22-32, mm/launch.cuh:105-183).
 * sfa and sfb are ignored. */
OG_API int32_t og_mm_launch(const OgGemm* g, const void* a, const void* b, const void* sfa,
                            const void* sfb, void* c, int32_t device, void* stream);

/* ---- block-scaled library: replaces opengemm/src/smm/capi.cu:6-32 -------- */

OG_API int32_t og_smm_abi(void);
OG_API const char* og_smm_error(void);
OG_API int32_t og_smm_kernels(void);
OG_API int32_t og_smm_kernel(int32_t i, OgGemm* out);
/* smm/launch.cuh:38-57 */
OG_API int32_t og_smm_bind(OgGemm* g);
/* sfa / sfb: scales in the 128x4 blocked layout (smm/launch.cuh:87-150, smm/tmap.cuh:21-36). */
OG_API int32_t og_smm_launch(const OgGemm* g, const void* a, const void* b, const void* sfa,
                             const void* sfb, void* c, int32_t device, void* stream);

/* ---- additions with no counterpart in the reference ----------------------- */

/* Output variant: besides the reference's fourteen dtype names, og_mm_bind accepts
 * "<format>.bf16" for every dense float format ("bf16.bf16", "f16.bf16", "tf32.bf16",
 * "e4m3.bf16", "e5m2.bf16", "e3m2.bf16", "e2m3.bf16", "e2m1.bf16", "e4m3xe5m2.bf16"):
 * same operands and tile plans, the f32 accumulator rounded to bfloat16 (nearest
 * even) on the way out, C a row-major bfloat16 [m, n]; and "<format>.f16" for the
 * same nine, C a row-major IEEE half [m, n].  og_mm_kernels / og_mm_kernel
 * enumerate the reference's formats only.
 *
 * Rasterisation: OgGemm.walk selects the order tiles are visited in, with the
 * reference's numbering (opengemm/src/mm/types.cuh:78-84): 0 bands `supergroup`
 * tiles wide along N; 1 the same, serpentine; 2 blocks inside a band; 3 a
 * generalised Hilbert curve; 4 bands along M.  Block-scaled formats, whose
 * reference struct carries no walk, use 0.
 *
 * Cluster-K: OgGemm.cluster_k = 2, 4 or 8 with use_2cta = 0 makes that many CTAs of one
 * thread-block cluster share every output tile, each taking a contiguous slice of K; the
 * slices' accumulators meet in the shared memory of the cluster's first CTA (distributed
 * shared memory, no trip through global memory), which stores the tile.  For shapes with
 * fewer tiles than SMs (small M, decode).  The reference's cluster_k planes add into a
 * zeroed C with atomics instead (opengemm/src/mm/kernel.cuh:29-36,86-96).  The request is
 * lowered to what fits: no more ways than K blocks, and the landing zone of
 * (cluster_k - 1) x tile width x 512 bytes must leave a three-stage ring. */

/* The native tile plan of a bound GEMM, for tuners and reports. */
typedef struct {
  int32_t cta_group; /* CTAs per MMA: 1 or 2 */
  int32_t tile_m, tile_n, block_k, stages;
  int32_t swap;      /* operands exchanged: B rows ride the 128-row MMA side */
  int32_t epi_staged; /* epilogue stages rows in shared memory and stores whole 128-byte lines */
  int32_t epi_tma;    /* ... and they leave by TMA store (32-bit output behind a long K loop) */
  int32_t acc_slots; /* accumulator buffers in tensor memory */
  int32_t tmem_cols, smem_bytes;
  int32_t tiles, grid; /* output tiles; CTAs launched */
  int32_t group;     /* rasterisation band width in tiles */
  int32_t stream_k;  /* partial wave cut along K across clusters (split_k >= 2) */
  int32_t use_clc;   /* tiles handed out by cluster launch control; grid = one cluster per tile */
  int32_t fixed_shape; /* served by a kernel compiled for exactly this tile shape (og_b200_set_fixed_kernels) */
  int32_t cluster_k; /* CTAs of a cluster sharing each tile along K (OgGemm.cluster_k with use_2cta = 0), else 1 */
  int32_t plain;     /* served by the build of the run-time-shaped kernel that has no optional feature compiled in */
} OgPlan;

/* Describe how `g` (already bound by og_mm_bind / og_smm_bind) would run on `device`
 * (pass -1 for "assume 148 SMs", which needs no GPU). */
OG_API int32_t og_b200_plan(const OgGemm* g, int32_t device, OgPlan* out);

/* Launch like og_mm_launch / og_smm_launch (chosen by g->dtype) with a device status
 * word: `status` points to a zero-initialised int32 in device-accessible memory.  A wait
 * that gives up stores (site | cta << 8) there instead of spinning forever; the kernel
 * then leaves through its ordinary teardown and the context stays usable.  Read the word
 * back after synchronising and hand it to og_b200_status. */
OG_API int32_t og_b200_launch_checked(const OgGemm* g, const void* a, const void* b,
                                      const void* sfa, const void* sfb, void* c, int32_t device,
                                      void* stream, int32_t* status);

/* Turns the status word of og_b200_launch_checked into a return code: OG_OK for 0,
 * else OG_ERR_TIMEOUT with og_mm_error() naming the wait (which role, which CTA). */
OG_API int32_t og_b200_status(int32_t status_word);

/* Launch like og_mm_launch / og_smm_launch (chosen by g->dtype) with every output
 * multiplied by `alpha` in float32 before it is stored (the product of per-tensor
 * dequantisation scales of fp8 / fp4 operands, for instance).  Float formats only:
 * s8 and u8 answer OG_ERR_LAUNCH. */
OG_API int32_t og_b200_launch_alpha(const OgGemm* g, const void* a, const void* b,
                                    const void* sfa, const void* sfb, void* c, int32_t device,
                                    void* stream, float alpha);

/* Output variant: C = alpha * (A . B^T) + bias, with `bias` a float32 device vector of
 * n values, one per column of C, added in float32 before the store (alpha = 1 adds the
 * bias only).  Float formats only.  The reference's epilogues store the bare product
 * (opengemm/src/mm/kernel.cuh:410-596, opengemm/src/smm/kernel.cuh:374-598). */
OG_API int32_t og_b200_launch_bias(const OgGemm* g, const void* a, const void* b,
                                   const void* sfa, const void* sfb, void* c, int32_t device,
                                   void* stream, float alpha, const void* bias);

/* Output variant: C leaves block-scaled - quantised along N exactly as the reference's
 * quantize (opengemm/python/quant.py:99-122) followed by to_blocked (quant.py:82-97) would
 * quantise a bfloat16 C - so that it can be the A operand of the next block-scaled GEMM
 * without a round trip through memory in bfloat16.  `out_format` is "nvfp4", "mxfp8" or
 * "mxfp4"; `c_packed` receives m x n/2 bytes (fp4) or m x n bytes (mxfp8), row-major;
 * `c_scales` the 128x4 blocked scales (ceil(m/128)*128 x ceil(n/(4*block))*4 bytes; rows past
 * m are left untouched).  g->dtype must be a block-scaled format or a "<format>.bf16" name;
 * n a multiple of 64, the tile width a multiple of 64, swap_ab 0.  The reference's
 * epilogues write bfloat16 or float32 only (opengemm/src/smm/kernel.cuh:374-598). */
OG_API int32_t og_b200_launch_quantized(const OgGemm* g, const void* a, const void* b,
                                        const void* sfa, const void* sfb, void* c_packed,
                                        void* c_scales, int32_t device, void* stream,
                                        const char* out_format);

/* Fused epilogue: z = alpha * (A . B^T) + bias is written to `preactivation` (if not
 * null), and C = activation(z) + residual.  All in float32, rounded once per tensor
 * written.  `residual` and `preactivation` are [m, n] row-major in C's type; `residual`
 * may be C itself, `preactivation` starts on a 16-byte boundary.  Float formats only.
 * With `out_format` the activation's value leaves block-scaled as in
 * og_b200_launch_quantized (no residual or pre-activation then).  Launches run the
 * static schedule without an operand swap: split_k, cluster_k, use_clc, walk and swap_ab
 * of `g` are not followed.  Up to four rows of 16-bit operands take a kernel of their own. */
typedef struct OgEpilogue {
  const void* bias;     /* float32 [n], or null */
  const void* residual; /* or null */
  void* preactivation;  /* or null */
  void* out_scales;     /* with out_format: the 128x4 blocked scales */
  float alpha;
  int32_t activation;   /* 0 none, 1 relu, 2 gelu, 3 gelu in its tanh form, 4 silu */
  int32_t out_format;   /* 0 C's own type, 1 nvfp4, 2 mxfp8, 3 mxfp4 */
} OgEpilogue;
OG_API int32_t og_b200_launch_fused(const OgGemm* g, const void* a, const void* b, const void* sfa,
                                    const void* sfb, void* c, int32_t device, void* stream,
                                    const OgEpilogue* epilogue);

/* Do now what launches on `device` do on first use: opt every kernel into its shared
 * memory and allocate the stream-K workspaces.  Call it before capturing launches into
 * a CUDA graph, or to keep the first request of a server free of allocations. */
OG_API int32_t og_b200_prepare_device(int32_t device);

/* The order a bound `g` visits its output tiles in: writes (M index, N index) pairs for
 * tile 0, 1, ... into `out` (room for `cap` integers) and returns the number of tiles,
 * or a negative status.  Needs no GPU. */
OG_API int32_t og_b200_tile_order(const OgGemm* g, int32_t* out, int32_t cap);

/* Testing aid.  The calling thread's next launch credits `bytes` more to each of its
 * stage barriers than its loads deliver, so the first wait for data runs out after the
 * limit of og_b200_set_wait_limit_ms and the launch reports it through its status word.
 * Nothing faults and nothing spins without bound. */
OG_API void og_b200_test_overcredit_next_launch(int32_t bytes);

/* The complete tile plan of a bound `g` for a device of `sm_count` SMs, as one JSON
 * object of integers written to `out` (what the standalone-kernel emitter bakes
 * into the code it writes).  Needs no GPU. */
OG_API int32_t og_b200_describe(const OgGemm* g, int32_t sm_count, char* out, int32_t cap);

/* Block-scaled quantisation on the GPU, the step upstream of every block-scaled GEMM:
 * `x` ([rows, k] bfloat16, or float32 when x_is_f32) -> `packed` (the operand in the
 * format's storage: k/2 bytes per row for nvfp4 / mxfp4, k for mxfp8), `scales`
 * ([rows, k/block] bytes, row-major; may be null) and `scales_blocked` (the 128x4
 * blocked layout og_smm_launch reads, ceil(rows/128)*128 x ceil(k/(4*block))*4 bytes;
 * may be null).  Same arithmetic, bit for bit, as the reference's torch helper
 * (opengemm/python/quant.py:99-122 followed by to_blocked, quant.py:82-97), in one
 * pass.  `format` is "nvfp4", "mxfp8" or "mxfp4".  Errors: og_b200_quantize_error(). */
OG_API int32_t og_b200_quantize(const char* format, const void* x, int32_t x_is_f32, int64_t rows,
                                int64_t k, void* packed, void* scales, void* scales_blocked,
                                int32_t device, void* stream);
OG_API const char* og_b200_quantize_error(void);

/* Launches use programmatic dependent launch: the next kernel of a stream may start
 * while this one drains.  By default every global-memory access of a kernel first
 * waits for the previous kernel to complete, so chained GEMMs (C of one feeding the
 * next) are safe.  With `yes` != 0 the caller vouches, process-wide, that no earlier
 * kernel in the stream writes the A / B / scale operands of a launch (weights and
 * inputs already resident, as in a benchmark loop): operand loads then start without
 * waiting, and only the stores wait - which is the only mode the reference has
 * (opengemm/src/mm/kernel.cuh:209,479-483).  Default 0. */
OG_API void og_b200_set_independent_inputs(int32_t yes);

/* Specialised builds of the kernel.  The hot tile shapes (pairs of CTAs on 256-row tiles,
 * the decode tile) also exist as kernels compiled for that one shape, with the plan's
 * constants folded in; and every variant exists once more with a run-time tile shape but
 * none of the optional features (stream-K, cluster launch control, cluster-K, bias, alpha,
 * half or block-scaled output, the non-default tile walks) compiled in, which is what a
 * launch that asks for none of them runs when no fixed-shape kernel matches its plan: a
 * GEMM of a tile or two per CTA runs its code once, from a cold instruction cache, and is
 * timed by the amount of code on its path.  All builds compute the same bits.  `yes` = 0
 * sends every launch to the full run-time kernel (default 1; the environment variable
 * OPENGEMM_FIXED=0 sets the default to 0). */
OG_API void og_b200_set_fixed_kernels(int32_t yes);

/* Limit of every device-side wait in milliseconds (default 2000).  Waits for a whole
 * accumulator, which sit behind a K loop of the others, allow twice as long. */
OG_API void og_b200_set_wait_limit_ms(int32_t ms);

/* No counterpart in the reference.  The same launch as og_mm_launch / og_smm_launch
 * (by g->dtype; bind `g` first) for callers that must not allocate device memory
 * inside a launch: processes that fixed their memory budget at start-up, code
 * running under an allocator that owns the rest of the GPU, latency-critical loops
 * that cannot absorb cudaMalloc's implicit device synchronisation.  It runs the
 * stream-K schedule out of a fixed workspace that is part of the library image
 * (about 18.5 MiB held by every GPU that loads the library, until exit) and calls
 * no allocating routine.  Limits: grids of at most 148 CTAs (a device needing more
 * partial-sum regions is refused with OG_ERR_LAUNCH and a message); one call at a
 * time per device, because all calls share the workspace: kernels of two calls
 * that overlap on the GPU race.  The first call on each device looks up the
 * workspace's address on that device; make it before any stream capture.
 * `error_text` (may be null) receives up to `error_text_cap` bytes on failure. */
OG_API int32_t og_b200_launch_no_alloc(const OgGemm* g, const void* a, const void* b,
                                       const void* sfa, const void* sfb, void* c, int32_t device,
                                       void* stream, char* error_text, int32_t error_text_cap);

/* ---- gradients of a product, and mixtures of experts: no counterpart in the reference ----
 *
 * Element types are 1 (bfloat16) and 2 (float16), for router logits also 0 (float32).
 * Activations are those of OgEpilogue, and the gated pairs 5 (silu(gate) * up) and
 * 6 (gelu(gate) * up), where gate and up are the first and the second half of the columns.
 * All calls are asynchronous on `stream`; none allocates or synchronises. */

/* A product whose rows fall into groups, each with a matrix of its own.
 *   mode 0  out[r] = act(alpha_e * x[r] . w_e^T)           x [rows, k], w [groups, n, k], out [rows, n] (gated: n/2)
 *   mode 1  out[r] = x[r] . w_e                            x [rows, n], w [groups, n, k], out [rows, k]
 *   mode 2  out[e] = sum over e's rows of x[r]^T w[r]      x [rows, n], w [rows, k],      out [groups, n, k]
 * Group e has the rows offsets[e] .. offsets[e + 1]; rows of `out` past the last group are
 * left as they were.  With `tokens` row r of mode 0's x is row tokens[r] of a [x_rows, k]
 * tensor.  dtype "bf16" or "f16", for mode 0 also "e4m3" (written as bfloat16).
 * Rows of all operands are multiples of 16 bytes and start on such boundaries.  A single
 * group needs no table: offsets may be null.  Errors: og_b200_experts_error(). */
typedef struct OgExpertProduct {
  const void* x;
  const void* w;
  const int32_t* offsets; /* device, [groups + 1], or null */
  const int32_t* tokens;  /* device, [rows], or null; mode 0 */
  const float* alpha;     /* device, [groups], or null; mode 0 */
  void* out;
  void* preactivation;    /* mode 0: [rows, n], the activation's argument, or null */
  int32_t mode, groups, rows, x_rows, n, k;
  int32_t activation;     /* mode 0 */
  int32_t out_f32;        /* modes 1 and 2: write float32 */
  float factor;           /* on every product, before the activation (beside alpha) */
  int32_t beside_previous; /* 1: the caller vouches that a launch of this call, over as many rows,
                              went to the stream before, that it writes nothing which this one
                              reads or writes, and that all of this one's memory was the
                              caller's before that launch; the two then run side by side */
  int32_t tile;           /* 0: chosen by an estimate; to measure or test one: 1 a pair of CTAs with
                             256 columns (not with `tokens`), 2 one CTA with 256, 3 with 128, 4 with 64 */
  char dtype[16];
} OgExpertProduct;
OG_API int32_t og_b200_expert_product(const OgExpertProduct* product, int32_t device, void* stream);
OG_API const char* og_b200_experts_error(void);

/* The choice of experts.  Scores are softmax (or logistic, `sigmoid`) values of the logits
 * [tokens, experts]; the choice is by score + bias (float32 [experts], or null), the lowest
 * index first among equals.  With groups > 1 only the `top_groups` groups of experts with
 * the largest sum of their best `group_top` (1 or 2) choice scores are open.  Weights
 * [tokens, top_k] are the chosen scores (divided by their sum if `renormalise`) times
 * `scale`.  A logit of -infinity is never chosen; a token with fewer than top_k experts
 * left has index -1 and weight 0 in the places that stay empty.  Errors: og_b200_routing_error(). */
typedef struct OgRoute {
  int64_t tokens;
  int32_t dtype, experts, top_k, sigmoid, groups, top_groups, group_top, renormalise;
  float scale;
} OgRoute;
OG_API int32_t og_b200_route(const OgRoute* route, const void* logits, const float* bias, float* weights,
                             int32_t* indices, int32_t device, void* stream);
/* Gradient of the logits (their type) for a gradient of the weights; `indices` as chosen. */
OG_API int32_t og_b200_route_gradient(const OgRoute* route, const float* grad_weights, const void* logits,
                                      const int32_t* indices, void* grad_logits, int32_t device, void* stream);

/* Order of the rows by expert, in the order of the (token, choice) pairs inside one.
 * offsets [experts + 1]: first row of each expert; token_of_row [tokens * top_k]; positions
 * [tokens, top_k]: the row of each pair, -1 where the index is outside 0 .. experts - 1
 * (then rows past offsets[experts] do not exist).  workspace: ceil(tokens * top_k / 8192) *
 * experts integers (null up to 8192 pairs). */
OG_API int32_t og_b200_expert_plan(const int32_t* indices, int64_t tokens, int32_t top_k, int32_t experts,
                                   int32_t* offsets, int32_t* token_of_row, int32_t* positions,
                                   int32_t* workspace, int32_t device, void* stream);

/* out[r] = x[token_of_row[r]] for the rows r < min(rows, *row_limit); rows of row_bytes, a
 * multiple of 16, on 16-byte boundaries. */
OG_API int32_t og_b200_expert_gather(const void* x, const int32_t* token_of_row, const int32_t* row_limit, void* out,
                                     int64_t row_bytes, int32_t rows, int32_t device, void* stream);

/* out[t] = residual[t] + sum over j of weights[t, j] * y[positions[t, j]] in float32, in the
 * order of j; weights null: ones; residual null: zero.  y [rows, n] of `dtype`, or float32
 * if y_is_f32; out and residual [tokens, n] of `dtype`. */
OG_API int32_t og_b200_expert_combine(int32_t dtype, int32_t y_is_f32, const void* y, const float* weights,
                                      const int32_t* positions, const void* residual, void* out, int64_t tokens,
                                      int32_t top_k, int32_t n, int32_t device, void* stream);
/* grad_y[positions[t, j]] = weights[t, j] * grad[t] (rows that no pair has are left as they
 * were) and grad_weights[t, j] = <grad[t], y[positions[t, j]]>, 0 where there is no row. */
OG_API int32_t og_b200_expert_combine_gradient(int32_t dtype, const void* grad, const void* y, const float* weights,
                                               const int32_t* positions, void* grad_y, float* grad_weights,
                                               int64_t tokens, int32_t top_k, int32_t n, int32_t device, void* stream);

/* dz = grad * act'(z) for rows [0, rows), or [0, min(rows, *row_limit)) if row_limit (device) is
 * given; other rows are neither read nor written and add nothing to the sums.
 * z, dz [rows, n]; grad [rows, n] (gated: n/2).  bias_gradient (float32 [n], or null; not for
 * a gated activation): column sums of dz before it is rounded, through a workspace of
 * ceil(rows / 16) * n floats.  Without an activation z and dz are not used. */
OG_API int32_t og_b200_activation_gradient(int32_t dtype, int32_t activation, const void* grad, const void* z, void* dz,
                                           float* bias_gradient, float* workspace, const int32_t* row_limit,
                                           int64_t rows, int32_t n, int32_t device, void* stream);
OG_API const char* og_b200_routing_error(void);

/* Gradients of C = act(factor * A . B^T + bias): with dz = grad * act'(z),
 *   grad_a = factor * dz . B,  grad_b = factor * dz^T . A,  grad_bias = column sums of dz.
 * grad and z [m, n] (z not used without an activation), a [m, k], b [n, k], all of `dtype`
 * ("bf16" or "f16"), n and k multiples of 8, on 16-byte boundaries; grad_a and grad_b of
 * `dtype` or float32 (out_f32), grad_bias float32 [n].  A gradient whose pointer is null is
 * not computed.  The 16-byte aligned workspace (dz, partial sums) holds at least what
 * og_b200_gemm_gradients_workspace answers for the same structure (workspace and
 * workspace_bytes aside); a negative answer is an error code.  Errors:
 * og_b200_experts_error(). */
typedef struct OgGemmGradients {
  const void *grad, *a, *b, *z;
  void *grad_a, *grad_b;
  float* grad_bias;
  void* workspace;
  int64_t workspace_bytes;
  int32_t m, n, k, activation, out_f32;
  float factor;
  char dtype[16];
} OgGemmGradients;
OG_API int32_t og_b200_gemm_gradients(const OgGemmGradients* g, int32_t device, void* stream);
OG_API int64_t og_b200_gemm_gradients_workspace(const OgGemmGradients* g, int32_t device);

#ifdef __cplusplus
}
#endif
#endif /* OPENGEMM_B200_H */
