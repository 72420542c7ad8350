/*
 * moe_mi355x.h — C ABI of the MI355X (gfx950) quantised MoE-layer library, libmoe_mi355x.so.
 *
 * The reference (Tigerly1/moe-lab) has no native FFI: its drop-in boundary is the Python "variant"
 * module contract (reference README.md:141-158, moelab/mlx_backend.py:3-8, moelab/torch_backend.py:3-5):
 *     prepare(w_gate, w_up, w_down) -> state;  run(state, x, idx, wts, act) -> y;  dequant(state)
 * plus run_slots (moelab/variants/mlx/metal_q4_moe.py:49-51) and the fused router tail topk_norm
 * (moelab/router.py:71-80). Each entry point below replaces the GPU work behind one of those calls;
 * the Python variant modules in moe-lab_amd/variants/ bind them with ctypes (moe-lab_amd/_lib.py).
 *
 * Conventions (all entry points):
 *   - every pointer is a device pointer (HBM), except the moe_experts_t descriptor itself, which
 *     lives in host memory and is read during the call only;
 *   - all work is enqueued on `stream` (a hipStream_t, passed as void*; NULL = default stream) and
 *     is asynchronous; nothing allocates device memory and nothing synchronises the host;
 *   - outputs and workspace are caller-allocated; sizes come from the *_workspace_bytes queries;
 *   - return 0 on success, a negative MOE_ERR_* code on invalid arguments (checked before any
 *     launch; mirrors the reference's shape asserts, e.g. metal_q4_moe.py:34) or launch failure;
 *   - reentrant; calls that share a workspace must be stream-ordered. The library's only mutable state is the table
 *     of moe_experts_run_static's array addresses, one per device, filled once under a lock (and that array).
 */
#ifndef MOE_MI355X_H
#define MOE_MI355X_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* return codes */
#define MOE_OK 0
#define MOE_ERR_ARG (-1)       /* shape, size or pointer argument invalid */
#define MOE_ERR_DTYPE (-2)     /* activation dtype or weight format not supported by this entry */
#define MOE_ERR_WORKSPACE (-3) /* workspace missing or smaller than *_workspace_bytes */
#define MOE_ERR_LAUNCH (-4)    /* the HIP runtime refused a launch */
#define MOE_ERR_ALIGN (-5)     /* a pointer is not 16-byte aligned */

/* activation / logits dtypes */
#define MOE_DTYPE_BF16 0
#define MOE_DTYPE_F16 1
#define MOE_DTYPE_F32 2

/*
 * Weight formats. The reference's state holds, per projection, codes u32 [E, N, K/8] (8 nibbles per word,
 * low nibble first) plus scales/biases bf16 [E, N, K/64] (int4 g64, metal_q4_decode_v4.py:161-169) or E8M0
 * bytes u8 [E, N, K/32] (MXFP4, metal_mxfp4_moe.py:448-455). This library takes the same numbers packed
 * row by row: each of the E*N rows is one record of moe_row_bytes(fmt, K) bytes, the row's K/2 code bytes
 * (the reference's words, unchanged) followed by its group metadata, zero-padded to a multiple of 16:
 *   MOE_FMT_INT4_G64: K/64 words, word g = scale_g (bf16, low half) | bias_g (bf16, high half) << 16
 *   MOE_FMT_MXFP4:    K/32 E8M0 bytes
 * so a row streams as one contiguous run. moelab_amd.formats converts in both directions.
 */
#define MOE_FMT_INT4_G64 0
#define MOE_FMT_MXFP4 1

/* GLU activations (reference metal_q4_decode_v4.py:36-41, metal_mxfp4_gptoss.py:36-43) */
#define MOE_ACT_SWIGLU 0      /* silu(g) * u */
#define MOE_ACT_GEGLU 1       /* tanh-GELU(g) * u (Gemma-4) */
#define MOE_ACT_GPTOSS 2      /* g = min(g,7), u = clip(u,-7,7), g * sigmoid(1.702 g) * (u + 1) */

/* activations of moe_linear */
#define MOE_LIN_NONE 0
#define MOE_LIN_SILU 1        /* z * sigmoid(z) */
#define MOE_LIN_GELU 2        /* tanh-GELU(z) */

/* expert-path selection for moe_experts_run */
#define MOE_PATH_AUTO 0       /* T == 1 -> per-slot GEMV (two launches); T > 1 -> grouped expert tiles */
#define MOE_PATH_SLOTS 1      /* per-slot GEMV over all T*k slots, no grouping, two launches (the stock-style
                                 gather of the reference's pre-tile kernels) */
#define MOE_PATH_GROUPED 2    /* grouped expert tiles: each selected expert's weights read once */

/* One projection of all E experts: N output rows of K inputs. */
typedef struct {
    const void* rows;    /* packed rows [E, N, moe_row_bytes(fmt, K)], 16-byte aligned */
    const float* bias;   /* optional additive row bias fp32 [E, N] (gpt-oss), NULL if none */
    const void* tiles;   /* optional: the same weights in the tile-major layout below (moe_tiles_pack of rows),
                            E * moe_tile_bytes(fmt, N, K) bytes, 16-byte aligned. The grouped path (T > 1)
                            streams these; NULL in any of gate/up/down: it reads rows (slower) */
} moe_proj_t;

/* Bytes of one packed row of K inputs in format fmt (0 for an invalid fmt or K). */
size_t moe_row_bytes(int fmt, int K);

/*
 * Tile-major layout (no counterpart in the reference, whose Metal kernels read its words row by row): the
 * grouped T > 1 path loads 16 rows x 128 inputs per MFMA step group, and HBM delivers such loads near its peak
 * only as contiguous bursts, so the same numbers are re-laid out once, at load time, on the device:
 *   tiles [E][N/16][S = ceil(K/128)][slice record], a slice record = 16 rows x 128 inputs:
 *     1024 bytes of code words: 16 bytes at offset 16 * (r + 16 g) (row r, lane group g = 0..3) hold the
 *     row's words (index within the row, s = slice)
 *         MOE_FMT_INT4_G64: 16s + 2g, 16s + 2g + 1, 16s + 8 + 2g, 16s + 9 + 2g
 *         MOE_FMT_MXFP4:    16s + g, 16s + 4 + g, 16s + 8 + g, 16s + 12 + g
 *     each with its nibbles (codes e0 .. e7, low nibble first) stored as e0 e2 e4 e6 e1 e3 e5 e7
 *     then the metadata of the slice's groups, per row r:
 *         MOE_FMT_INT4_G64: 8 bytes at 1024 + 8r = group words 2s, 2s + 1, each (scale, bias) times 2^-X
 *                           (bf16, exact), X the row's exponent below   (record: 1152 bytes)
 *         MOE_FMT_MXFP4:    4 bytes at 1024 + 4r = E8M0 bytes of groups 4s .. 4s + 3   (record: 1088 bytes)
 *     words and groups past K (K % 128 == 64) are zero.
 *   int4 only, after the records of all E experts: row exponents int8 [E][N]. X = (biased exponent of the row's
 *     largest bf16 |scale| or |bias|) - 137, i.e. floor(log2 of it) - 10, clamped to [-120, 120]; 0 for an
 *     all-zero row or one holding an inf or NaN. The scaled metadata puts every row's largest at [2^10, 2^11), so
 *     the kernels that dequantise to fp16 keep any absolute scale range (scales of 1e-8 or 1e30 alike); the tile
 *     kernels multiply each row's sums by 2^X.
 * moe_tile_bytes: bytes per expert of an N x K projection in this layout (int4: records + N exponent bytes;
 *                 0 if N % 16, K % 64 or fmt invalid).
 * moe_tiles_pack: rows [E, N, moe_row_bytes(fmt, K)] -> tiles [E * moe_tile_bytes(fmt, N, K)], on `stream`.
 */
size_t moe_tile_bytes(int fmt, int N, int K);
int moe_tiles_pack(int fmt, int E, int N, int K, const void* rows, void* tiles, void* stream);

/* Expert weights: gate/up [E, F, d], down [E, d, F]. */
typedef struct {
    int32_t fmt;         /* MOE_FMT_* */
    int32_t E, d, F;
    moe_proj_t gate, up, down;
} moe_experts_t;

/*
 * Fused router: gate GEMV + router tail.
 * Replaces the stock gate GEMV self.gate(x) (reference e2e.py:57-59) followed by router.topk_norm
 * (reference moelab/router.py:71-80; semantics router.py:1-12).
 *   x [T, d] bf16, wr [E, d] bf16, bias [E] fp32 or NULL
 *   logits [T, E] fp32 out: x . wr^T (+ bias), fp32, fixed reduction order (see the kernel source)
 *   idx [T, k] int32, wts [T, k] fp32 out; norm = 1: softmax over the top-k logits (= renormalised
 *   softmax), norm = 0: full-softmax probabilities (DeepSeek-V2 greedy); weights are multiplied by scale.
 *   Ties: lowest expert id. NaN logits count as -inf. Limits: E <= 1024, 1 <= k <= min(E, 32), d % 8 == 0.
 *   Two launches: the logits over many workgroups, then the tails, one wave per token. counters: unused (may be NULL; kept, with moe_router_counter_count, so existing callers link
 *   unchanged).
 */
int moe_router(const void* x, const void* wr, const float* bias, int T, int d, int E, int k, int norm, float scale,
               float* logits, int32_t* idx, float* wts, int32_t* counters, void* stream);
int moe_router_counter_count(int T);

/*
 * Fused router that also builds the slot grouping: moe_router's logits launch, then one launch that runs every token's
 * tail (one wave per token: the same ids and weights as moe_router), after which the last workgroup to finish sorts
 * the T*k slots p = t*k + j stably by expert, with the counts' offsets from a wave prefix sum. Replaces the stock gate
 * GEMV +
 * router.topk_norm (as moe_router) followed by the grouping prepass of the grouped kernels (reference
 * metal_q4_tiles_v2.py:362-373 MAP kernel order, closed form of reference triton_fused_moe.py:56-70 align()).
 *   x, wr, bias, T, d, E, k, norm, scale, logits, idx, wts: as moe_router;
 *   counts [E], offsets [E+1], sorted [T*k], active [E], meta [2] int32 out: as moe_group (meta[1] = 0).
 */
int moe_router_group(const void* x, const void* wr, const float* bias, int T, int d, int E, int k, int norm,
                     float scale, float* logits, int32_t* idx, float* wts, int32_t* counts, int32_t* offsets,
                     int32_t* sorted, int32_t* active, int32_t* meta, void* stream);

/*
 * Router tail on given logits: reference moelab/router.py:71-80 topk_norm(logits, k, norm).
 *   logits [T, E] of dtype MOE_DTYPE_*; idx [T, k] int32, wts [T, k] fp32 out.
 */
int moe_topk(const void* logits, int dtype, int T, int E, int k, int norm, float scale, int32_t* idx, float* wts,
             void* stream);

/*
 * Slot grouping: slots p = t*k + j sorted stably by expert (reference metal_q4_tiles_v2.py:362-373 MAP
 * kernel order; closed form of reference triton_fused_moe.py:56-70 align()).
 *   idx [n] int32 in, n <= 0x78000000; counts [E], offsets [E+1], sorted [n], active [E], meta [2] int32 out.
 *   meta[0] = number of experts with count > 0 (listed ascending in active[0..meta[0]) , rest -1);
 *   meta[1] = number of slots whose id is outside [0, E) (they join no group).
 */
int moe_group(const int32_t* idx, int n, int E, int32_t* counts, int32_t* offsets, int32_t* sorted, int32_t* active,
              int32_t* meta, void* stream);

/*
 * Expert part of the layer: reference variant run(state, x, idx, wts, act) (metal_q4_moe.py:54-64,
 * metal_mxfp4_moe.py:474-512, metal_mxfp4_gptoss.py:129-167):
 *   y[t] = residual[t] + sum_j wts[t,j] * ( down_e( act(gate_e x_t + bg_e, up_e x_t + bu_e) ) + bd_e ),
 *   e = idx[t,j]; residual optional (NULL = 0).
 *   x [T, d] of x_dtype (MOE_DTYPE_BF16, MOE_DTYPE_F16 or MOE_DTYPE_F32: fp16 and fp32 x enter the gate/up
 *   products exactly, as 2 or 3 bf16 planes whose sum is x; the reference's fp32 path is its exact scalar tiles,
 *   metal_q4_moe.py:62-64); y and residual [T, d] of y_dtype (any of the three; the reference returns x.dtype,
 *   MOE_DTYPE_F32 gives the unrounded result); idx [T, k] int32; wts [T, k] fp32.
 *   path: MOE_PATH_*; nored = 1 writes the unweighted per-slot outputs y[T*k, d] instead (reference
 *   run_slots / NORED, metal_q4_moe.py:49-51; per-slot path only, residual must be NULL).
 *   Accumulation in fp32; the GLU output h is kept between the two launches as an unevaluated sum of two
 *   bf16 planes (about 16 significant bits, where the reference kernels store it in x.dtype). Exception: int4
 *   grouped calls with more than 16 slots per expert on average (prefill-sized T, path MOE_PATH_GROUPED with
 *   the tile-major copies) run the down projection, and above 32 also the gate/up, on fp16 MFMA: weights
 *   rounded once to fp16 from the row-exponent-scaled metadata, x and h carried as fp16 with a power-of-two
 *   exponent per row (no overflow and no flush to zero whatever a row's absolute scale); within a row, weights
 *   more than 2^13 below the row's largest |16 s|, |b| fall into fp16's subnormal range (absolute step 2^-19 of
 *   the row's largest |s|, |b|); ~1e-3 of the outputs' RMS in the worst case measured, 1.4e-3 with one scale
 *   group per row at 256x the others' (numpy emulation). From 17 to 32 slots per expert the down does the
 *   same where its grid fills the chip (row blocks of 128 x passes of 128 slots >= 256), else both stages stay on exact
 *   codes. Before such a down, from 21 slots per expert, the gate/up (bf16 or fp16 x) also runs on fp16 MFMA, on the
 *   exact weights s (q - 8) and x in that fp16 form, with b + 8 s applied to the group sums of x: the call's error
 *   against 64 bits is that of the exact-code gate/up before the same down.
 *   Requirements: d % 64 == 0, F % 64 == 0, F <= 16384; x, y, rows 16-byte aligned.
 *   workspace: moe_experts_workspace_bytes(...) bytes (any contents; every call writes what it reads). Calls
 *   sharing a workspace must be stream-ordered. With the tile-major copies a grouped call whose x (T d 2 bytes) or h
 *   (T k F 2 bytes) passes 2^32 - 4096 bytes runs as equal blocks of tokens, each with a part of the workspace.
 */
int moe_experts_run(const moe_experts_t* w, const void* x, int x_dtype, const int32_t* idx, const float* wts, int T,
                    int k, int act, int path, int nored, void* y, int y_dtype, const void* residual, void* workspace,
                    size_t workspace_bytes, void* stream);
size_t moe_experts_workspace_bytes(const moe_experts_t* w, int T, int k, int path);

/*
 * moe_experts_run without a workspace argument: no counterpart in the reference. For callers that cannot
 * allocate (code under HIP graph capture, serving loops or harnesses that forbid allocation): the workspace is a
 * device array inside the library, MOE_STATIC_SCRATCH_BYTES on each GPU it runs on, held until the process ends.
 * Arguments, results and errors as moe_experts_run; calls whose workspace (moe_experts_workspace_bytes) exceeds
 * MOE_STATIC_SCRATCH_BYTES return MOE_ERR_WORKSPACE before any launch (the Qwen3-30B-A3B shape fits calls of up
 * to 110 tokens).
 * It allocates nothing. Every call on one GPU uses that GPU's one array, which keeps the last call's contents (no
 * call needs particular contents): calls that overlap on one GPU (other streams, other threads) race, and the
 * caller must order them. The first call on each device (the device of `stream`; the current device for the null
 * stream) looks up the array's address (hipGetSymbolAddress); make it outside graph capture: a call with T = 0 does
 * only that.
 */
#define MOE_STATIC_SCRATCH_BYTES ((size_t)32 << 20)
int moe_experts_run_static(const moe_experts_t* w, const void* x, int x_dtype, const int32_t* idx, const float* wts,
                           int T, int k, int act, int path, int nored, void* y, int y_dtype, const void* residual,
                           void* stream);

/*
 * The same call split at the one data dependency inside it, the GLU output h held in the workspace.
 * The reference dispatches these as separate kernels as well (metal_q4_decode_v4.py:177-184 _k1 gate_up,
 * _k2 down). stages = MOE_STAGE_GATE_UP: grouping (grouped path) + gate/up + GLU, h into the workspace;
 * MOE_STAGE_DOWN: down projection + combine from the h a previous GATE_UP call with the same arguments
 * left in the same workspace (stream-ordered); MOE_STAGE_ALL = both = moe_experts_run. Lets a caller
 * interleave other work between the two stages, or time each stage on its own stream.
 */
#define MOE_STAGE_GATE_UP 1
#define MOE_STAGE_DOWN 2
#define MOE_STAGE_ALL 3
int moe_experts_run_stages(const moe_experts_t* w, const void* x, int x_dtype, const int32_t* idx, const float* wts,
                           int T, int k, int act, int path, int nored, void* y, int y_dtype, const void* residual,
                           void* workspace, size_t workspace_bytes, int stages, void* stream);

/*
 * Router and experts in one call: moe_router's logits (same fixed order, so the same ids) and tail, then
 * moe_experts_run's default path. The reference calls them one after the other, the stock gate GEMV, router.topk_norm,
 * then the variant's run (reference e2e.py:57-64, moelab/router.py:71-80).
 *   T == 1: the router launch computes the logits only and every gate/up wave runs the tail over the 128..1024 logits
 *   itself for its own slot (no hand-off between workgroups inside a launch: measured at 1-2 us per round trip on this
 *   part); one wave writes idx / wts.
 *   T > 1: the router's two launches (as moe_router_group) compute the logits, run the tails and build the slot
 *   grouping and the expert kernels' pass lists, so the expert launches follow with no top-k or grouping launch of
 *   their own; where the gate/up wave tiles group the slots in-kernel (a few slots per expert) they do it there
 *   instead (one of their workgroups writes the lists for the down stage).
 *   x [T, d] bf16 (MOE_DTYPE_BF16 only: the gate GEMV reads bf16); wr [E, d] bf16, wr_bias [E] fp32 or NULL;
 *   norm, scale: as moe_router; idx [T, k] int32 and wts [T, k] fp32 out (as moe_router's); y, residual, act,
 *   y_dtype: as moe_experts_run. workspace: moe_layer_workspace_bytes(w, T, k) bytes (any contents).
 */
int moe_layer_run(const moe_experts_t* w, const void* x, int x_dtype, const void* wr, const float* wr_bias, int T,
                  int k, int norm, float scale, int act, int32_t* idx, float* wts, void* y, int y_dtype,
                  const void* residual, void* workspace, size_t workspace_bytes, void* stream);
size_t moe_layer_workspace_bytes(const moe_experts_t* w, int T, int k);

/*
 * moe_layer_run with S shared experts (the caller semantics of the reference's model patches, routed experts then the
 * shared module: e2e.py:57-68 Qwen-style gated shared expert, e2e.py:138-147 DeepSeek-V2): w holds E = E_r + S experts
 * as for moe_experts_run_shared (experts E_r .. E_r + S - 1 the shared ones), wr [E_r, d] routes over the first E_r.
 *   y[t] = residual[t] + sum_j wts[t,j] * expert_{idx[t,j]}(x_t) + g_t * sum_s expert_{E_r + s}(x_t),
 *   g_t = sigmoid(x_t . gate) (gate: bf16 [d], computed by the router launch as one more logit row, in the logits'
 *   fixed order) or 1 when gate is NULL. The router's launches write idx / wts [T, k] (the routed slots), the merged
 *   [T, k + S] slot lists and, at T > 1, their grouping; then the experts as moe_experts_run_shared.
 *   Limits: 1 <= S < E, E_r <= 1024, k <= min(E_r, 32), k + S <= 64.
 *   workspace: moe_layer_shared_workspace_bytes(w, S, T, k) bytes (any contents).
 */
int moe_layer_run_shared(const moe_experts_t* w, int S, const void* x, int x_dtype, const void* wr,
                         const float* wr_bias, const void* gate, int T, int k, int norm, float scale, int act,
                         int32_t* idx, float* wts, void* y, int y_dtype, const void* residual, void* workspace,
                         size_t workspace_bytes, void* stream);
size_t moe_layer_shared_workspace_bytes(const moe_experts_t* w, int S, int T, int k);

/*
 * Shared experts: S always-on experts added to every token, the caller semantics of the reference's model
 * patches (reference e2e.py:66-68 Qwen-style gated shared expert, sigmoid(x . w_gate) * shared_expert(x);
 * e2e.py:146-147 DeepSeek, + shared_experts(x)). The reference runs them as stock mlx-lm modules; here they go
 * through the same expert kernels as the routed experts:
 *   y[t] = residual[t] + g_t * sum_s ( down_s( act(gate_s x_t + bg_s, up_s x_t + bu_s) ) + bd_s ),
 *   g_t = sigmoid(x_t . gate) (gate: bf16 [d], fp32 dot in a fixed order) or 1 when gate is NULL.
 *   ws: the S shared experts as an expert set (E = S <= 32; same formats, packing and optional tile copies).
 *   x, y, residual, dtypes, act: as moe_experts_run (path auto: per-slot GEMV at T == 1, grouped tiles above).
 *   workspace: moe_shared_experts_workspace_bytes(ws, T) bytes (any contents), as for moe_experts_run.
 * A layer with routed and shared experts is moe_experts_run (routed, into y) followed by this call with
 * residual = y.
 */
int moe_shared_experts_run(const moe_experts_t* ws, const void* x, int x_dtype, int T, int act, const void* gate,
                           void* y, int y_dtype, const void* residual, void* workspace, size_t workspace_bytes,
                           void* stream);
size_t moe_shared_experts_workspace_bytes(const moe_experts_t* ws, int T);

/*
 * Routed and shared experts in one call (no counterpart in the reference, whose model patches run the shared
 * experts as a separate module after the routed ones, e2e.py:66-68 and 146-147): w holds E = E_r + S experts,
 * experts E_r .. E_r + S - 1 being the shared ones (same d, F, format and packing as the routed ones: the two
 * sets' rows concatenated, with tile copies packed over all E). Token t's slots are its k routed slots (idx, wts
 * as moe_experts_run; ids outside [0, E_r) join no group) followed by the S shared slots, expert E_r + s with
 * weight g_t = sigmoid(x_t . gate) (gate: bf16 [d]) or 1 when gate is NULL:
 *   y[t] = residual[t] + sum_j wts[t,j] * expert_{idx[t,j]}(x_t) + g_t * sum_s expert_{E_r + s}(x_t),
 * the experts and path as in moe_experts_run. One grouping, one combine, and the shared experts' work inside
 * the routed launches (the two-call form costs a second grouping, combine and slot-list launch, and runs the few
 * shared experts on grids too small to fill the chip). Limits: 1 <= S < E, k >= 1, k + S <= 64.
 *   workspace: moe_experts_shared_workspace_bytes(w, S, T, k, path) bytes (any contents).
 */
int moe_experts_run_shared(const moe_experts_t* w, int S, const void* x, int x_dtype, const int32_t* idx,
                           const float* wts, int T, int k, int act, int path, const void* gate, void* y, int y_dtype,
                           const void* residual, void* workspace, size_t workspace_bytes, void* stream);
size_t moe_experts_shared_workspace_bytes(const moe_experts_t* w, int S, int T, int k, int path);

/*
 * Read-bandwidth probe of the timing harness's contention guard (the reference's guard times a read-bound reduction,
 * moelab/guard.py:31-45): MOE_PROBE_SINK workgroups stream src [nbytes] (16-byte aligned, nbytes % 16 == 0) with
 * 16-byte loads, the expert kernels' weight-load pattern, and nothing else; workgroup b writes the XOR of the 32-bit
 * words it read to sink[b] (so the XOR of sink [MOE_PROBE_SINK] uint32 is the XOR of the buffer's words).
 */
#define MOE_PROBE_SINK 1024
int moe_probe_read(const void* src, size_t nbytes, uint32_t* sink, void* stream);

/*
 * Products grouped by expert, 16-bit weights (the reference multiplies quantised experts only; its unquantised form is the
 * per-expert loop of moelab/variants/cuda/torch_loop.py:11-17). Slots p = 0 .. M - 1 are sorted by group: group e holds
 * offsets[e] <= p < offsets[e + 1] (offsets [E + 1] int32 on the device, offsets[0] = 0; values outside [0, M] are
 * clamped). offsets NULL: one group of all M slots (E = 1).
 *   moe_grouped_mm:    y[p][n]     = sum_k x[r(p)][k] w[e][n][k] (+ bias[e][n]),  r(p) = rows[p], or p when rows is NULL
 *   moe_grouped_mm_dx: dx[p][k]    = sum_n dy[r(p)][n] w[e][n][k]
 *   moe_grouped_mm_dw: dw[e][n][k] = sum_p dy[dy_idx[p]][n] x[x_idx[p]][k],  dbias[e][n] = sum_p dy[dy_idx[p]][n]
 *                      (groups without a slot: zeros; a NULL index list: the slot itself)
 * Operands and bias are of one type, MOE_DTYPE_BF16 or MOE_DTYPE_F16; the result is of that type, rounded once from fp32
 * sums in a fixed order, or MOE_DTYPE_F32 (dbias: the operands' type). x [x_rows, K] with ldx elements from row to row
 * (dy alike); w [E, N, K], results and bias contiguous. Slots behind the last group are left as they were, or set to zero
 * with fill = 1. An index outside its matrix reads as a row of zeros.
 * Requirements: M <= 0x7fffff00, E <= 1024, N % 8 == 0, K % 8 == 0, strides % 8 == 0, N, K <= 2^20, strides <= 2^21; pointers
 * 16-byte aligned; a matrix read through an index list (for dw: either, then both) at most 0xB0000000 bytes.
 */
int moe_grouped_mm(const void* x, const void* w, const void* bias, const int32_t* offsets, const int32_t* rows, int64_t M,
                   int64_t x_rows, int64_t ldx, int E, int N, int K, int dtype, void* y, int y_dtype, int fill,
                   void* stream);
int moe_grouped_mm_dx(const void* dy, const void* w, const int32_t* offsets, const int32_t* rows, int64_t M,
                      int64_t dy_rows, int64_t lddy, int E, int N, int K, int dtype, void* dx, int dx_dtype, int fill,
                      void* stream);
int moe_grouped_mm_dw(const void* dy, const void* x, const int32_t* offsets, const int32_t* dy_idx, const int32_t* x_idx,
                      int64_t M, int64_t dy_rows, int64_t lddy, int64_t x_rows, int64_t ldx, int E, int N, int K, int dtype,
                      void* dw, int dw_dtype, void* dbias, void* stream);

/*
 * One product with its epilogue: y = act(x w^T + bias) + residual, x [T, K] (ldx elements from row to row), w [N, K],
 * bias [N], residual and y [T, N]; types, alignment and sizes as moe_grouped_mm; act: MOE_LIN_*. The sums, bias, activation
 * and residual are fp32, rounded once. z [T, N] (or NULL): the sums with bias before the activation, in the operands' type,
 * what moe_linear_act_bwd takes. residual may be y. Gradients: dz = dy act'(z) by moe_linear_act_bwd (dz = dy without an
 * activation), then dx [T, K] = dz w by moe_linear_dx, and dw [N, K] = dz^T x and dbias [N] (or NULL), the sums of dz's
 * columns, by moe_linear_dw, in the operands' type; lddz and ldx: elements from row to row.
 * workspace: the call's _workspace_bytes(T, N, K), any contents (0: NULL will do). With few output tiles the sums are split
 * into parts, whose results are added in a fixed order.
 */
size_t moe_linear_workspace_bytes(int64_t T, int N, int K);
size_t moe_linear_dx_workspace_bytes(int64_t T, int N, int K);
size_t moe_linear_dw_workspace_bytes(int64_t T, int N, int K);
int moe_linear_dx(const void* dz, const void* w, int64_t T, int64_t lddz, int N, int K, int dtype, void* dx, void* workspace,
                  size_t workspace_bytes, void* stream);
int moe_linear_dw(const void* dz, const void* x, int64_t T, int64_t lddz, int64_t ldx, int N, int K, int dtype, void* dw,
                  void* dbias, void* workspace, size_t workspace_bytes, void* stream);
int moe_linear(const void* x, const void* w, const void* bias, const void* residual, int act, int64_t T, int64_t ldx, int N,
               int K, int dtype, void* y, int y_dtype, void* z, void* workspace, size_t workspace_bytes, void* stream);
/* z [T, N] in 16 bits, or NULL and its 8-bit form codes, scales (moe_act8_pack). */
int moe_linear_act_bwd(const void* dy, int64_t lddy, const void* z, const void* codes, const void* scales, int act, int64_t T,
                       int N, int dtype, void* dz, void* stream);

/*
 * Activations kept in 8 bits for a backward pass. Rows of C values (C % 32 == 0) as int8 codes [M, C] and one exponent byte
 * per 32 neighbours, scales [M, C / 32]: value = code * 2^(scale - 133), |code| <= 127, a rounding of at most half a step.
 * scale = biased exponent of the block's largest magnitude, one more if that would round to 128 (254 at most: there the
 * code stays 127); 255: the block holds an infinity or NaN and reads as NaN.
 *   moe_act8_pack, _unpack: 16-bit values to that form, and back (to bf16, fp16 or fp32; into the type they came from it is
 *                           exact, but for 65536, the form of fp16 values from 65280 on, which becomes fp16's 65504).
 *   moe_glu_fwd: gu [M, 2 F] (gate columns, then up; ldgu elements from row to row) -> h [M, F] = act(gate, up) and, codes not
 *                NULL, gu's 8-bit form (codes [M, 2 F], scales [M, 2 F / 32]). act: MOE_ACT_*; F % 32 == 0.
 *   moe_glu_bwd: from that form (or gu itself with codes NULL), dh [M, F] (16-bit or MOE_DTYPE_F32) and row weights wts [M]
 *                (NULL: 1): dgu [M, 2 F] = wts dh act'(gate, up), hw [M, F] = wts h (or NULL), dwts [M] = sum_f dh h (or
 *                NULL). Where an act-2 clamp holds, the gradient is 0.
 */
int moe_act8_pack(const void* x, int64_t ldx, int64_t M, int C, int dtype, void* codes, void* scales, void* stream);
int moe_act8_unpack(const void* codes, const void* scales, int64_t M, int C, void* out, int dtype, void* stream);
int moe_glu_fwd(const void* gu, int64_t ldgu, int64_t M, int F, int act, int dtype, void* h, void* codes, void* scales,
                void* stream);
int moe_glu_bwd(const void* codes, const void* scales, const void* gu, int64_t ldgu, const void* dh, int dh_dtype,
                const float* wts, int64_t M, int F, int act, int dtype, void* dgu, void* hw, float* dwts, void* stream);

/*
 * The expert layer on 16-bit weights, forward and backward (the unquantised form of moe_experts_run; reference
 * moelab/variants/cuda/torch_loop.py:11-17, which has no backward pass):
 *   y[t] = residual[t] + sum_j wts[t][j] w_down[e] . act(w_gate_up[e] . x[t]),  e = idx[t][j]
 * w_gate_up [E, 2 F, d] (gate rows, then up), w_down [E, d, F]; x, residual [T, d] and the weights of m->dtype, y too or
 * MOE_DTYPE_F32; idx [T, k] int32 (a slot with an id outside [0, E) adds nothing), wts [T, k] fp32.
 * h is rounded to the 16-bit type between the launches; the GLU takes the gate/up sums, and the sum over slots their rows, in fp32.
 *   keep [moe_mlp_keep_bytes]: the slots' grouping, which the backward pass reads; written in every case.
 *   gu [T k, 2 F], or codes [T k, 2 F] and scales [T k, F / 16]: what the backward pass needs of the gate/up rows, in 16 or in
 *   8 bits (forward: each may be NULL; backward: one of the two forms).
 *   moe_mlp_bwd: dx [T, d], dwts [T, k] fp32, dw_gate_up, dw_down (as the weights), each may be NULL. dwts of slots with an id
 *   outside [0, E) is left as it was. From the kept 8-bit values, gradients are those of the function at these values.
 * Requirements: E <= 1024, d % 8 == 0, F % 32 == 0, T d and 2 F d at most 0x58000000, T k <= 0x78000000; pointers 16-byte
 * aligned. workspace: any contents; forward and backward sizes from their queries. moe_mlp_bwd takes T > 0.
 */
typedef struct {
    int32_t E, d, F, act, dtype;
    const void* w_gate_up;
    const void* w_down;
} moe_mlp_t;
size_t moe_mlp_keep_bytes(const moe_mlp_t* m, int T, int k);
size_t moe_mlp_fwd_workspace_bytes(const moe_mlp_t* m, int T, int k);
size_t moe_mlp_bwd_workspace_bytes(const moe_mlp_t* m, int T, int k);
int moe_mlp_fwd(const moe_mlp_t* m, const void* x, const int32_t* idx, const float* wts, int T, int k, const void* residual,
                void* y, int y_dtype, void* keep, void* gu, void* codes, void* scales, void* workspace, size_t workspace_bytes,
                void* stream);
int moe_mlp_bwd(const moe_mlp_t* m, const void* x, const float* wts, const void* dy, int T, int k, const void* keep, const void* gu,
                const void* codes, const void* scales, void* dx, float* dwts, void* dw_gate_up, void* dw_down, void* workspace,
                size_t workspace_bytes, void* stream);

/*
 * Routing by scores and groups (the reference's router is the softmax top-k of moe_topk, moelab/router.py:1-66; it leaves
 * group-limited gates to the stock module, e2e.py:129-150):
 *   s = sigmoid(logit) or softmax(logits) (MOE_SCORE_*); an expert ranks by s + bias[e], without a bias by its logit;
 *   groups > 1: experts E / groups * g ... form group g, its value is the largest ranking value in it (MOE_GROUP_MAX) or the sum
 *   of the two largest (MOE_GROUP_TOP2; without a bias the scores'); the top_groups groups of largest value stay;
 *   idx [T, k]: the k experts of largest ranking value in the groups that stay, of equals the lowest id first (groups alike);
 *   wts [T, k] fp32 = scale s, with norm scale s / (sum of the k experts' s) (0 where that is 0; a softmax's from the chosen
 *   logits alone).
 * A NaN logit counts as -inf. Experts whose logit is -inf or whose ranking value is -inf or NaN are chosen after all others,
 * lowest id first, with weight 0. Scores and their sums are fp64: of two experts the better one is chosen also where fp32
 * scores are equal.
 *   moe_topk_scored: logits [T, E] of dtype MOE_DTYPE_*, contiguous.
 *   moe_topk_scored_bwd: dlogits [T, E] of the logits' type from dwts [T, k] fp32 and the call's idx; the bias and the choice
 *   have no gradient.
 *   moe_router_scored: moe_router's logits x . wr^T + wr_bias (x [T, d], wr [E, d] bf16, wr_bias [E] fp32 or NULL; logits
 *   [T, E] fp32 out), then moe_topk_scored.
 * Requirements: E <= 1024, groups <= 64, E % groups == 0, k <= min(32, top_groups E / groups); MOE_GROUP_TOP2: groups of 2
 * experts at least.
 */
#define MOE_SCORE_SOFTMAX 0
#define MOE_SCORE_SIGMOID 1
#define MOE_GROUP_MAX 0
#define MOE_GROUP_TOP2 1
typedef struct {
    int32_t E, k, score, groups, top_groups, group_score, norm;
    float scale;
    const float* bias;   /* [E] fp32 or NULL */
} moe_scored_t;
int moe_topk_scored(const moe_scored_t* r, const void* logits, int dtype, int T, int32_t* idx, float* wts, void* stream);
int moe_topk_scored_bwd(const moe_scored_t* r, const void* logits, int dtype, int T, const int32_t* idx, const float* dwts,
                        void* dlogits, void* stream);
int moe_router_scored(const moe_scored_t* r, const void* x, const void* wr, const float* wr_bias, int T, int d, float* logits,
                      int32_t* idx, float* wts, void* stream);

/*
 * MXFP4 operands made on the device, and their products (the reference multiplies MXFP4 weights by 16-bit activations inside
 * its expert kernels only, metal_mxfp4_moe.py). A matrix of `rows` rows and K columns (K % 32 == 0):
 *   codes  [rows, K / 2]: an E2M1 code per element, two to a byte, the low half first (the packed words of MOE_FMT_MXFP4);
 *   scales [ceil(K / 256), rows, 8]: byte 4 (b % 2) + b / 2 of (s, row) is the E8M0 exponent of columns 256 s + 32 b .. + 31, 127
 *   past K.
 * value = e2m1(code) 2^(byte - 127); 255 is NaN. `matrices` of them follow each other, codes and scales alike; the scales'
 * buffer has moe_mx4_scale_bytes(matrices, rows, K) bytes (8 per row and step, and 16 that are read but not used).
 *   moe_mx4_quantize: x (bf16, fp16 or fp32; ldx elements between rows, = K with several matrices). byte = biased exponent of
 *       the block's largest magnitude less 2; codes to nearest, ties to even, past 6 to 6; a zero keeps its sign. Blocks below
 *       2^-124 become zeros of byte 0, blocks with an infinity or NaN codes of 0 and byte 255. (formats.py's rule.)
 *   moe_mx4_dequantize: the values, to bf16, fp16 or fp32, rounded to nearest (bf16, fp32: exact but below 2^-126).
 *   moe_mx4_linear: y = act(x w^T + bias) + residual with w [N, K] in that form, and x either 16-bit rows [T, K] (ldx; then xc
 *       and xs receive its form, or are NULL) or, x NULL, its form xc, xs. bias [N], residual and z [T, N] of `dtype`, bf16 or
 *       fp16 (x's type); y of dtype or MOE_DTYPE_F32; act, z, workspace as moe_linear.
 *   moe_mx4_grouped_mm: moe_grouped_mm on w [E, N, K] and x [x_rows, K] in that form (x alike: 16-bit rows, or its form). For the
 *       workspace: has_form, xc and xs are given.
 *   moe_mx4_linear_dx, moe_mx4_grouped_mm_dx: dx = dz w with w's values as `dtype` numbers (fp16: rounded to it), dz [T, N] (dy
 *       [M, N]) of `dtype`, as moe_linear_dx and moe_grouped_mm_dx without an index list.
 *   moe_mx4_linear_bwd: the gradients of moe_mx4_linear that are wanted (dx [T, K], dw [N, K], db [N]; any NULL): dz = dy act'(z) in
 *       `dtype` (act MOE_LIN_NONE: dy itself, z not read), dx = dz w, dw = dz^T x at the values of xc, xs (needed for dw) and
 *       wc, ws (for dx).
 *   moe_mx4_bias_grad: db [E, N] of `dtype` = the sums of dy's rows by group (moe_grouped_mm's groups; offsets NULL with E = 1):
 *       the gradient of a bias beside frozen weights. A group without rows: zeros.
 * Products of codes and powers of two are exact, their sums fp32; bias, activation and residual fp32, rounded once.
 * Requirements: K % 32 == 0, N % 8 == 0, K, N <= 2^20, rows <= 0x7fffff00, ldx % 8 == 0 and <= 2^21, E <= 1024; pointers 16-byte
 * aligned; x_rows K / 2 <= 0xB0000000 with an index list.
 */
size_t moe_mx4_scale_bytes(int64_t matrices, int64_t rows, int K);
int moe_mx4_quantize(const void* x, int64_t ldx, int64_t matrices, int64_t rows, int K, int dtype, void* codes, void* scales,
                     void* stream);
int moe_mx4_dequantize(const void* codes, const void* scales, int64_t matrices, int64_t rows, int K, void* out, int dtype,
                       void* stream);
size_t moe_mx4_linear_workspace_bytes(int64_t T, int N, int K);
int moe_mx4_linear(const void* x, int64_t ldx, void* xc, void* xs, const void* wc, const void* ws, const void* bias,
                   const void* residual, int act, int64_t T, int N, int K, int dtype, void* y, int y_dtype, void* z,
                   void* workspace, size_t workspace_bytes, void* stream);
size_t moe_mx4_linear_dx_workspace_bytes(int64_t T, int N, int K);
int moe_mx4_linear_dx(const void* dz, int64_t lddz, const void* wc, const void* ws, int64_t T, int N, int K, int dtype, void* dx,
                      void* workspace, size_t workspace_bytes, void* stream);
int moe_mx4_grouped_mm_dx(const void* dy, int64_t lddy, const void* wc, const void* ws, const int32_t* offsets, int64_t M, int E,
                          int N, int K, int dtype, void* dx, int dx_dtype, int fill, void* stream);
size_t moe_mx4_linear_bwd_workspace_bytes(int64_t T, int N, int K, int act, int dx, int dw, int db);
int moe_mx4_linear_bwd(const void* dy, int64_t lddy, const void* z, int act, const void* xc, const void* xs, const void* wc,
                       const void* ws, int64_t T, int N, int K, int dtype, void* dx, void* dw, void* db, void* workspace,
                       size_t workspace_bytes, void* stream);
size_t moe_mx4_bias_grad_workspace_bytes(int64_t M, int E, int N);
int moe_mx4_bias_grad(const void* dy, int64_t lddy, const int32_t* offsets, int64_t M, int E, int N, int dtype, void* db,
                      void* workspace, size_t workspace_bytes, void* stream);
size_t moe_mx4_grouped_mm_workspace_bytes(int64_t M, int64_t x_rows, int E, int K, int has_form);
int moe_mx4_grouped_mm(const void* x, int64_t ldx, void* xc, void* xs, int64_t x_rows, const void* wc, const void* ws,
                       const void* bias, const int32_t* offsets, const int32_t* rows, int64_t M, int E, int N, int K, int dtype,
                       void* y, int y_dtype, int fill, void* workspace, size_t workspace_bytes, void* stream);

/* Library version and build target, for logs. */
const char* moe_version(void);

#ifdef __cplusplus
}
#endif
#endif /* MOE_MI355X_H */
