/*
 * mxfa.h - C ABI of the MI355X (gfx950) flash-attention training path.
 *
 * Drop-in for the host wrappers and kernels of the 02-flash-attention crate of
 * glaucomaa/mx230. Every entry point below names the reference interface it
 * replaces (paths relative to the reference repository).
 *
 * Conventions
 *   - Plain C types only: device pointers are `void*` / `float*` obtained from
 *     hipMalloc (or any allocator of device memory); `stream` is a
 *     hipStream_t passed as `void*` (NULL = the null stream).
 *   - Layouts (row-major, contiguous):
 *       Q, O, dO, dQ : [B][Hq][N][d]
 *       K, V, dK, dV : [B][Hkv][N][d]
 *       LSE, Delta   : [B][Hq][N]  (always fp32; LSE in natural-log units)
 *     With B = Hq = Hkv = 1 and d = 64 this is exactly the reference's
 *     [N][64] layout (attention_flash.cu:17-89).
 *     Query head h reads KV head h / (Hq / Hkv) (grouped-query attention,
 *     03-llm-engine/src/cpu.rs:194,224); dK / dV of a KV head are the sum
 *     over the query heads that share it.
 *   - dtype MXFA_F32: every tensor above is fp32. dtype MXFA_BF16: Q, K, V,
 *     O, dO, dQ, dK, dV are bf16 (raw uint16 storage), LSE and Delta fp32,
 *     and all accumulation is fp32.
 *   - All launches are asynchronous on `stream`. The run_* entry points never
 *     synchronise and never allocate device memory. The library's own state
 *     is the one-launch backward's: a static 4 MB array of Delta flags per
 *     device, a launch counter (epoch), the counter of mxfa_bwd_delta_fallbacks
 *     and the settings of mxfa_set_bwd_options. Launches in flight together
 *     on one device are safe (see mxfa_bwd_one_launch); ordering is the
 *     caller's stream order.
 *   - The roofline and measurement probes are declared in mxfa_probes.h.
 *   - Errors are returned as negative codes (see mxfa_status); nothing aborts
 *     and no C++ exception crosses this boundary. The reference panics on a
 *     launch failure (02-flash-attention/src/main.rs:87,122,142,172,204,209).
 *   - Device pointers must be 16-byte aligned.
 */
#ifndef MXFA_H
#define MXFA_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    MXFA_OK = 0,
    MXFA_ERR_NULL = -1,        /* a required pointer is NULL */
    MXFA_ERR_SHAPE = -2,       /* B, Hq, Hkv, N, d or Hq % Hkv invalid */
    MXFA_ERR_DTYPE = -3,       /* unknown dtype */
    MXFA_ERR_UNSUPPORTED = -4, /* valid shape, but no kernel (e.g. d not in {64, 128}) */
    MXFA_ERR_ALIGN = -5,       /* a device pointer is not 16-byte aligned */
    MXFA_ERR_LAUNCH = -6,      /* the HIP runtime rejected a launch */
    MXFA_ERR_DEVICE = -7,      /* no usable gfx950 device */
    MXFA_ERR_WORKSPACE = -8,   /* a workspace smaller than mxfa_{bwd,prefill,prefill_batch,prefill_batch_mx}_workspace_bytes */
    MXFA_ERR_CODE_OBJECT = -9, /* the gfx950 code object is missing, malformed, for another
                                  processor, or lacks a kernel */
    MXFA_ERR_SCRATCH = -10     /* mxfa_run_bwd_noalloc: the shape needs more than
                                  mxfa_bwd_noalloc_scratch_bytes() */
} mxfa_status;

typedef enum { MXFA_F32 = 0, MXFA_BF16 = 1 } mxfa_dtype;

typedef struct {
    int B;        /* batch */
    int Hq;       /* query heads */
    int Hkv;      /* key/value heads; Hq % Hkv == 0 */
    int N;        /* sequence length (queries = keys) */
    int d;        /* head dim: 64 or 128 */
    int causal;   /* 0 or 1: key j visible to query i iff j <= i (main.rs:218) */
    int dtype;    /* mxfa_dtype */
    float scale;  /* softmax scale; 0 selects 1/sqrt(d) (main.rs:214) */
} mxfa_shape;

/* Library version as MAJOR*10000 + MINOR*100 + PATCH. */
int mxfa_version(void);

/* Human-readable text of a status code (static storage). */
const char *mxfa_strerror(int status);

/* The kernels are not part of libmxfa.so: they are one gfx950 code object,
 * mxfa_gfx950.hsaco (built by hipcc beside the library), loaded per device with
 * hipModuleLoadData and launched by name. */

/* Checks that `device` exists and is a gfx950 (MI355X), makes it current and
 * loads the code object on it (MXFA_ERR_CODE_OBJECT if that fails).
 * Optional: the run_* entry points load it on the current device at their
 * first launch there, and return MXFA_ERR_CODE_OBJECT if they cannot.
 * Replaces CudaContext::new(0) + load_kernels / load_bwd, which load the PTX
 * modules and look the kernels up by name
 * (02-flash-attention/src/main.rs:392-415, 514). */
int mxfa_init(int device);

/* Unloads the code object from every device it was loaded on (each device's
 * work must have completed); a later launch loads it again. */
int mxfa_shutdown(void);

/* Sets the code object file later loads read (NULL: mxfa_gfx950.hsaco in the
 * directory of libmxfa.so). Devices that already loaded one keep it until
 * mxfa_shutdown. Returns MXFA_OK; the file is checked when loaded.
 * Replaces the PTX paths the reference's build.rs exports to the crate
 * (kernel-build/src/lib.rs:37-55, :89-115). */
int mxfa_set_code_object(const char *path);

/* Checks a code object file on the host, with no device access (NULL: the
 * file later loads read): present and readable, a 64-bit little-endian ELF for
 * EM_AMDGPU with the AMDGPU HSA OS/ABI, built for gfx950. MXFA_OK or
 * MXFA_ERR_CODE_OBJECT. The counterpart of load_ptx's guard against an empty
 * stub module (common/src/lib.rs:11-18). */
int mxfa_check_code_object(const char *path);

/* Validates a shape exactly as every run_* entry point does; no GPU access. */
int mxfa_check_shape(const mxfa_shape *shape);

/* Forward, O only.
 * Replaces run_flash (02-flash-attention/src/main.rs:68-88) and kernel
 * attn_flash (02-flash-attention/kernels/attention_flash.cu:91-94). */
int mxfa_run_flash(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                   void *o, void *stream);

/* Forward, O and the per-row log-sum-exp L_i = m_i + ln(l_i).
 * Replaces run_flash_lse (main.rs:102-123) and attn_flash_lse
 * (attention_flash.cu:97-100, LSE at :85-87). */
int mxfa_run_flash_lse(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                       void *o, float *lse, void *stream);

/* Delta_i = sum_x dO[i][x] * O[i][x] (fp32 accumulation).
 * Replaces run_preprocess (main.rs:126-143) and attn_bwd_preprocess
 * (attention_bwd.cu:32-44). */
int mxfa_run_preprocess(const mxfa_shape *shape, const void *dout, const void *o, float *delta,
                        void *stream);

/* dQ pass only (overwrites dQ; atomic-free).
 * Replaces the attn_bwd_dq launch of run_bwd_flash (main.rs:202-204,
 * attention_bwd.cu:96-158). */
int mxfa_run_bwd_dq(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                    const void *dout, const float *lse, const float *delta, void *dq,
                    void *stream);

/* dK/dV pass only (overwrites dK, dV; atomic-free; with Hq > Hkv the sum over
 * the query heads of a group is done inside the kernel).
 * Replaces the attn_bwd_dkv launch of run_bwd_flash (main.rs:206-209,
 * attention_bwd.cu:165-243). */
int mxfa_run_bwd_dkv(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                     const void *dout, const float *lse, const float *delta, void *dk,
                     void *dv, void *stream);

/* The tiled backward: dK/dV pass then dQ pass, same stream, outputs
 * overwritten (no zeroing needed).
 * Replaces run_bwd_flash (02-flash-attention/src/main.rs:179-210). */
int mxfa_run_bwd_flash(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                       const void *dout, const float *lse, const float *delta, void *dq,
                       void *dk, void *dv, void *stream);

/* dQ pass that also computes Delta = rowsum(dO * O) for its query rows and
 * writes it to `delta` (the preprocess launch, attention_bwd.cu:32-44,
 * folded into the attn_bwd_dq launch, :96-158). */
int mxfa_run_bwd_dq_delta(const mxfa_shape *shape, const void *q, const void *k, const void *v, const void *o,
                          const void *dout, const float *lse, float *delta, void *dq, void *stream);

/* The whole backward from O in two launches, or one (below): the dQ pass
 * computes Delta = rowsum(dO * O) itself (writing it to `delta`, B*Hq*N fp32,
 * which the caller owns as for mxfa_run_preprocess) and the dK/dV pass reads it.
 * Replaces the sequence run_preprocess + run_bwd_flash (main.rs:126-143,
 * :179-210; attention_bwd.cu:32-44, :96-243) with the preprocess launch folded
 * into the dQ pass; results equal that sequence's up to the summation order of
 * Delta. */
int mxfa_run_bwd(const mxfa_shape *shape, const void *q, const void *k, const void *v, const void *o,
                 const void *dout, const float *lse, float *delta, void *dq, void *dk, void *dv,
                 void *stream);

/* 1 if mxfa_run_bwd and mxfa_run_bwd_ws run the dQ and dK/dV work of this
 * shape in one launch (for a GQA split through a workspace, the adding of the
 * split's partial sums included), else 0 (a dQ launch and a dK/dV launch, or
 * an invalid shape).
 * The one-launch form (bf16, d = 64 or 128) runs the dQ work-groups first;
 * they publish Delta per 128-row query block, and the dK/dV work-groups of the
 * same launch wait for the blocks they need. Each wait is bounded in time
 * (mxfa_bwd_options.delta_wait_us): after it the work-group computes those
 * Delta rows from O and dO itself, with the same arithmetic as the dQ
 * work-groups, so the results equal the two-launch form's bitwise either way.
 * mxfa_bwd_options.one_launch = 0 selects two launches, and so does a stream
 * under graph capture (a replayed launch would reuse the capture's flag
 * epoch); this query answers for an ordinary stream. An fp32 grid that fits the
 * GPU about at once also takes one launch unless one_launch = 0 or an output
 * shares memory with an input (the dK/dV work-groups compute Delta themselves,
 * in the dQ work's order, with no flags, captured or not, so the results equal
 * the two launches' bitwise); this query is 0 for it.
 * No counterpart in the reference: it tells callers (and benchmarks) which
 * kernels the backward from O (main.rs:126-143, :179-210) becomes. */
int mxfa_bwd_one_launch(const mxfa_shape *shape);

/* Process-wide settings of the one-launch backward, read at every launch
 * (default {1, 200, 2000000}). Meant for tests and measurement; settings changed while
 * other threads launch take effect at their next launch.
 * No counterpart in the reference (its backward is always two launches,
 * main.rs:179-210). */
typedef struct {
    int one_launch;    /* 1: one launch where available (bf16); 0: always two */
    int delta_wait_us; /* bound of each Delta wait in microseconds; < 0: never
                          wait, always compute Delta in the dK/dV work-group */
    int reduce_wait_us; /* bound of each wait of a GQA split's reduce work-
                           group for its shares, microseconds, >= 0 (see
                           mxfa_bwd_reduce_timeouts) */
} mxfa_bwd_options;
int mxfa_set_bwd_options(const mxfa_bwd_options *options);
int mxfa_get_bwd_options(mxfa_bwd_options *options);

/* Delta blocks (64 query rows of one head) that the one-launch backward's
 * dK/dV work-groups computed themselves on the current device, because their
 * wait ran out, since the library was loaded. A synchronous device-to-host
 * copy: call it after the launches of interest have completed. 0 in normal
 * operation; a count does not change results (see mxfa_bwd_one_launch). */
int mxfa_bwd_delta_fallbacks(unsigned long long *count);

/* Work-groups of the one-launch backward that add a GQA split's partial sums
 * and whose wait for them ran out, on the current device since the library
 * was loaded (a synchronous device-to-host copy, as above). Those work-groups
 * run after all of the split's work-groups have been dispatched, so the wait
 * ends in normal operation and the count stays 0; a count means the dK and dV
 * rows of those work-groups were written as NaN. The wait is bounded
 * (mxfa_bwd_options.reduce_wait_us, default 2 s) so that a launch always
 * ends.
 * No counterpart in the reference (no GQA, and its backward is two launches,
 * main.rs:179-210). */
int mxfa_bwd_reduce_timeouts(unsigned long long *count);

/* Bytes of device workspace the _ws entry points below can use (0 for an
 * invalid shape). dQ is a separate atomic-free pass and needs none. With GQA
 * (Hq > Hkv), when the key blocks alone would leave the GPU underfilled, the
 * dK/dV pass splits the work of each key block (its group's query heads, each
 * from the diagonal) over several work-groups, a causal block with more
 * queries over more of them: each writes fp32 partial dK/dV sums to the
 * workspace, and they are added in a fixed order (deterministic, atomic-free)
 * by the last work-groups of the one-launch backward, else by a second
 * launch. The size is 2 * planes * B * Hkv * N * d * 4 bytes, planes being
 * the most work-groups any key block takes, then 8 bytes per work-group of
 * the split (the flags by which the one-launch backward's adding work-groups
 * learn that a share's sums are written: each launch writes its own value,
 * so the workspace needs no clearing); 0 when no split helps (always without
 * GQA). A call uses its workspace until it completes: calls in flight at the
 * same time need their own.
 * The reference has no GQA (d = 64, one head, attention_bwd.cu:165-243); this
 * sizes the scratch of its dK/dV pass generalised to GQA groups. */
size_t mxfa_bwd_workspace_bytes(const mxfa_shape *shape);

/* mxfa_run_bwd_dkv with a caller-owned workspace (16-byte aligned, at least
 * mxfa_bwd_workspace_bytes(shape) bytes, else MXFA_ERR_ALIGN or
 * MXFA_ERR_WORKSPACE). workspace == NULL is allowed and runs the unsplit pass
 * (= mxfa_run_bwd_dkv). Results equal the unsplit pass's up to the summation
 * order over the query heads of a group; the workspace holds nothing the
 * caller needs afterwards.
 * Replaces the attn_bwd_dkv launch (attention_bwd.cu:165-243, main.rs:206-209)
 * for GQA shapes. */
int mxfa_run_bwd_dkv_ws(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                        const void *dout, const float *lse, const float *delta, void *dk,
                        void *dv, void *workspace, size_t workspace_bytes, void *stream);

/* mxfa_run_bwd with a caller-owned workspace for its dK/dV pass (as
 * mxfa_run_bwd_dkv_ws; NULL = mxfa_run_bwd).
 * Replaces run_preprocess + run_bwd_flash (main.rs:126-143, :179-210) as
 * mxfa_run_bwd does. */
int mxfa_run_bwd_ws(const mxfa_shape *shape, const void *q, const void *k, const void *v, const void *o,
                    const void *dout, const float *lse, float *delta, void *dq, void *dk, void *dv,
                    void *workspace, size_t workspace_bytes, void *stream);

/* mxfa_run_bwd_ws without a workspace argument and without allocating: the
 * split dK/dV pass keeps its fp32 partial sums and share flags in a static
 * device array of the library, mxfa_bwd_noalloc_scratch_bytes() (65 MiB) per
 * device, held from the
 * library's set-up on the device (mxfa_init, else this entry point's first
 * call there) until the process ends. Shapes whose mxfa_bwd_workspace_bytes
 * exceed it return MXFA_ERR_SCRATCH before any device work. No hipMalloc,
 * hipFree or other allocating call; the array needs no clearing (every call
 * overwrites what it reads). All calls on one device share the array and
 * keep the last call's contents, so calls that overlap on one device race
 * (serialise them, e.g. on one stream); results equal mxfa_run_bwd_ws's.
 * No counterpart in the reference: it is for callers that cannot allocate
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * allocation). */
int mxfa_run_bwd_noalloc(const mxfa_shape *shape, const void *q, const void *k, const void *v, const void *o,
                         const void *dout, const float *lse, float *delta, void *dq, void *dk, void *dv,
                         void *stream);
size_t mxfa_bwd_noalloc_scratch_bytes(void);

/* Naive backward baseline: one thread per query row, dK/dV scattered with
 * atomic adds. fp32 only. dQ, dK, dV MUST be zeroed by the caller.
 * Replaces run_bwd_naive (main.rs:147-173) and attn_bwd_naive
 * (attention_bwd.cu:48-90). */
int mxfa_run_bwd_naive(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                       const void *dout, const float *lse, const float *delta, void *dq,
                       void *dk, void *dv, void *stream);

/* Bytes of the N x N fp32 score scratch mxfa_run_naive_fwd needs
 * (B * Hq * N * N * 4). */
size_t mxfa_naive_scratch_bytes(const mxfa_shape *shape);

/* Naive forward baseline that materialises the scores: S = QK^T * scale
 * (masked to -inf above the diagonal when causal), row softmax in place,
 * O = S V. fp32 only; `s` holds mxfa_naive_scratch_bytes bytes.
 * Replaces Naive::run (main.rs:32-66) and attn_scores / attn_softmax /
 * attn_av (attention_naive.cu:8-70). */
int mxfa_run_naive_fwd(const mxfa_shape *shape, const void *q, const void *k, const void *v,
                       float *s, void *o, void *stream);

/* ---- Inference-side forward (prefill): token-major rows over a KV cache.
 * Replaces `attn_prefill` (03-llm-engine/kernels/llm.cu:3806-3815, body
 * :3674-3804; launched by gpu.rs:3235-3289): query row i of this chunk sits at
 * absolute position pos0 + i and attends to cache rows 0 .. pos0 + i (causal
 * with a diagonal offset). Q row i holds head h at elements
 * [h * head_dim, (h + 1) * head_dim) of a row q_stride elements long (the
 * fused QKV row in the reference); the K and V caches hold position j in rows
 * kv_stride elements long, KV head h / (n_head / n_kv_head) at
 * [kvh * head_dim, ...); the output row i likewise with out_stride. Rows
 * 0 .. pos0 + n_tok - 1 of both caches must be filled (the reference copies
 * the chunk's own K/V in first, copy_kv_batch at llm.cu:3635). Generalisations: bf16 as well
 * as fp32, head_dim 128 (bf16), any scale; the reference is fp32, head_dim 64,
 * scale 1/8. No LSE is written. */
typedef struct {
    int n_tok;      /* query rows of this chunk */
    int n_head;     /* query heads */
    int n_kv_head;  /* KV heads; n_head % n_kv_head == 0 */
    int head_dim;   /* 64 (fp32, bf16) or 128 (bf16) */
    int pos0;       /* absolute position of query row 0 */
    int q_stride;   /* elements between query rows (>= n_head * head_dim) */
    int kv_stride;  /* elements between cache rows (>= n_kv_head * head_dim) */
    int out_stride; /* elements between output rows (>= n_head * head_dim) */
    int dtype;      /* mxfa_dtype */
    float scale;    /* 0 -> 1/sqrt(head_dim) */
} mxfa_prefill_shape;

/* MXFA_OK if the prefill shape is supported; strides whose rows would not start
 * on 16-byte boundaries give MXFA_ERR_ALIGN, and pos0 + max(n_tok, n_head)
 * above 2^31 - 129 gives MXFA_ERR_SHAPE (a single row runs its GQA group's
 * heads as rows at positions pos0, pos0 + 1, ...). */
int mxfa_check_prefill(const mxfa_prefill_shape *shape);
int mxfa_run_prefill(const mxfa_prefill_shape *shape, const void *q, const void *kcache, const void *vcache,
                     void *out, void *stream);

/* The prefill over a paged KV cache. Replaces `attn_prefill_paged`
 * (03-llm-engine/kernels/llm.cu:3827-3836, body :3674-3804 with
 * PAGED = true; launched by gpu.rs:3270-3289): the same as mxfa_run_prefill,
 * except that logical cache position t sits in cache row
 * block_table[t / block_size] * block_size + t % block_size (kv_row<true>,
 * llm.cu:959-963), rows kv_stride elements apart from kcache / vcache.
 * block_table: int32 on the device, entries for positions 0 .. pos0 + n_tok - 1,
 * each a physical block inside the caches (not checked: a bad entry reads
 * outside them, as in the reference). block_size: a power of two (the
 * reference engine's KV_BLOCK is 16, gpu.rs:209); others give
 * MXFA_ERR_UNSUPPORTED. Outputs are bitwise those of mxfa_run_prefill over the
 * gathered, contiguous cache. */
int mxfa_run_prefill_paged(const mxfa_prefill_shape *shape, const void *q, const void *kcache, const void *vcache,
                           void *out, const int *block_table, int block_size, void *stream);

/* The prefill with its keys split over work-groups, for chunks whose query
 * blocks alone would leave most of the GPU idle (a few hundred tokens after a
 * long history, or a single decode-like row). Replaces the same
 * `attn_prefill` launch as mxfa_run_prefill (llm.cu:3806-3815, gpu.rs:3235-3289),
 * which has no counterpart of the split: each work-group takes a range of the
 * cache's 64-key stages of one 64-query block and writes its unnormalised
 * output and its rows' running max and sum to `workspace` (fp32); a second
 * launch adds the ranges (out = sum_s w_s O_s / sum_s w_s l_s with
 * w_s = 2^(m_s - max m)). Same arguments as mxfa_run_prefill, plus the
 * workspace: mxfa_prefill_workspace_bytes(shape) bytes, 16-byte aligned,
 * device memory (no contents needed; calls that share one race). When that
 * size is 0 the shape needs no split and this is mxfa_run_prefill (workspace
 * may be NULL). A smaller workspace gives MXFA_ERR_WORKSPACE, except that a
 * shape that gains from many ranges (one token far into a long context, an
 * fp32 chunk) takes a smaller one, or none, down to what 64-query blocks take
 * (at most 32 ranges), and uses as many as it holds. Results equal
 * mxfa_run_prefill's to fp32 rounding of the merge, not bitwise. */
size_t mxfa_prefill_workspace_bytes(const mxfa_prefill_shape *shape);
int mxfa_run_prefill_ws(const mxfa_prefill_shape *shape, const void *q, const void *kcache, const void *vcache,
                        void *out, void *workspace, size_t workspace_bytes, void *stream);
/* mxfa_run_prefill_paged with the same key split (replaces the
 * `attn_prefill_paged` launch, llm.cu:3827-3836, gpu.rs:3270-3289): the
 * paged cache arguments of mxfa_run_prefill_paged and the workspace of
 * mxfa_run_prefill_ws, sized by mxfa_prefill_workspace_bytes(shape) (the
 * same for both caches). Outputs are bitwise those of mxfa_run_prefill_ws over
 * the gathered, contiguous cache. */
int mxfa_run_prefill_paged_ws(const mxfa_prefill_shape *shape, const void *q, const void *kcache,
                              const void *vcache, void *out, const int *block_table, int block_size,
                              void *workspace, size_t workspace_bytes, void *stream);

/* ---- Rotary positions. Pair i of a head's first rotary_dim elements, (x1, x2)
 * = (x[i], x[i + rotary_dim / 2]) or, interleaved, (x[2i], x[2i + 1]), turns by
 * a = position * frequencies[i] (radians; the product is formed in 64 bits):
 *     y1 = factor (x1 cos a - x2 sin a),  y2 = factor (x2 cos a + x1 sin a);
 * the other elements are copied. inverse = 1 turns by -a with the same factor:
 * the transpose, which takes the gradients of the outputs to the inputs'. */
typedef struct {
    int B, Hq, Hkv, N; /* heads of Q and of K; Hkv = 0: Q alone */
    int head_dim;      /* a multiple of 8, at most 256 */
    int rotary_dim;    /* even, 2 .. head_dim */
    int interleaved;   /* 0 or 1 */
    int inverse;       /* 0 or 1 */
    int dtype;         /* mxfa_dtype */
    int pos0;          /* without positions: token n is at pos0 + n */
    float factor;      /* multiplies cosines and sines (1: a plain rotation) */
    /* strides in elements between batches, heads and tokens, of Q, K and their
     * outputs; rows are contiguous and start on 16-byte boundaries. Dimensions
     * of one element have no stride (any value). Outputs' strides are >= 0. */
    long long q_bs, q_hs, q_ts, k_bs, k_hs, k_ts;
    long long qo_bs, qo_hs, qo_ts, ko_bs, ko_hs, ko_ts;
    long long pos_bs; /* positions: elements between batches (0: shared) */
} mxfa_rotary_shape;
int mxfa_check_rotary(const mxfa_rotary_shape *shape);
/* One launch for Q and K. positions: int32 on the device, N per batch, any
 * sign; NULL: pos0 + n. frequencies: rotary_dim / 2 doubles on the device.
 * An output may be its own input (the same pointer and strides); one whose
 * span overlaps its input's otherwise gives MXFA_ERR_UNSUPPORTED, and Q and K
 * outputs must not overlap each other or the other's input (not checked: they
 * may be columns of the same rows). */
int mxfa_run_rotary(const mxfa_rotary_shape *shape, const void *q, const void *k, void *q_out, void *k_out,
                    const int *positions, const double *frequencies, void *stream);

/* ---- A batch of sequences over a paged KV cache. Sequence s has the rows
 * cu_q[s] .. cu_q[s + 1] - 1 of the batch's new tokens (cu_q[0] = 0; int32 on
 * the device, n_seq + 1 of them) and lens[s] positions in all, the new ones
 * the last: its i-th new token is at lens[s] - (cu_q[s + 1] - cu_q[s]) + i.
 * Position t's K and V are in cache row block_table[s * table_stride + t /
 * block_size] * block_size + t % block_size. The device arrays are read when
 * the kernels run, so a captured launch follows what they hold at each replay.
 * Nothing outside the buffers is accessed whatever they hold: rows past n_tok,
 * positions past the table and blocks outside the pool are left out when
 * written; when read, such a block counts as the nearest one in the pool and
 * positions past the table as not there, and the sequence's outputs are then
 * not specified. Rows past cu_q[n_seq] are left as they were. */
typedef struct {
    int n_tok;        /* rows of q / qkv and of the output */
    int n_seq;        /* sequences */
    int max_q;        /* attention: at least the most new tokens of a sequence;
                         rows past it are left as they were */
    int n_head, n_kv_head, head_dim;
    int block_size;   /* tokens per block, a power of two */
    int n_blocks;     /* blocks in the caches */
    int max_blocks;   /* entries of a block_table row */
    int table_stride; /* elements between block_table rows, >= max_blocks */
    int q_stride;     /* elements between rows of q / qkv */
    int kv_stride;    /* elements between cache rows */
    int out_stride;   /* elements between output rows */
    int dtype;        /* mxfa_dtype */
    float scale;      /* attention: 0 -> 1/sqrt(head_dim) */
} mxfa_batch_shape;
/* As mxfa_run_prefill_batch checks it. */
int mxfa_check_batch(const mxfa_batch_shape *shape);

/* Attention of the batch's new tokens over the cache: the token at position t
 * of its sequence attends to the positions 0 .. t (K and V of the new tokens
 * included, as mxfa_run_cache_append writes them). Query row r holds head h at
 * elements [h * head_dim, (h + 1) * head_dim), a cache row KV head h, the
 * output row likewise; head_dim 64 (fp32, bf16) or 128 (bf16). A row that sees
 * no position (a token at a negative one) is zeros, its lse -infinity; one whose
 * every seen score is -infinity has no softmax: NaN, its lse -infinity. lse:
 * NULL, or n_tok x n_head floats. A position that a row does not see never
 * reaches it, whatever its K and V hold. The workspace
 * (mxfa_prefill_batch_workspace_bytes, 16-byte aligned, no contents needed) is
 * used until the call completes: calls that may overlap need their own. The
 * key ranges of long sequences are joined in a fixed order: equal calls give
 * equal bits. out may be q (the same pointer and stride) or other columns of the
 * same rows; where it lies over q otherwise, or out, lse or the workspace over a
 * cache, q or each other, the call is refused (MXFA_ERR_UNSUPPORTED). */
size_t mxfa_prefill_batch_workspace_bytes(const mxfa_batch_shape *shape);
int mxfa_run_prefill_batch(const mxfa_batch_shape *shape, const void *q, const void *kcache, const void *vcache,
                           void *out, float *lse, const int *block_table, const int *cu_q, const int *lens,
                           void *workspace, size_t workspace_bytes, void *stream);

/* The cache append: row r of qkv holds token r's n_head query heads, then its
 * n_kv_head key heads, then its value heads; Q turns into q_out row r, K turns
 * into kcache and V is copied into vcache, at the rows of the tokens'
 * positions. rotary_dim = 0 (frequencies NULL): copies only. head_dim as for
 * mxfa_rotary_shape. q_out may be qkv (the same pointer and stride), or other
 * columns of the same rows; where it lies over qkv otherwise the call is refused
 * (MXFA_ERR_UNSUPPORTED). Any other overlap is the caller's to avoid. A token at
 * a negative position is left out, its q_out row too; one past the table has its
 * q_out row only. */
typedef struct {
    int rotary_dim, interleaved;
    float factor;
    const double *frequencies; /* device, rotary_dim / 2 */
} mxfa_append_rotary;
int mxfa_run_cache_append(const mxfa_batch_shape *shape, const mxfa_append_rotary *rotary, const void *qkv,
                          void *q_out, void *kcache, void *vcache, const int *block_table, const int *cu_q,
                          const int *lens, void *stream);

/* ---- A microscaled cache: the paged cache in 8 or 4 bits a value. Of each head's
 * row, 32 neighbouring elements share a power of two 2^(E - 127), one byte E;
 * an element is a code of `bits` bits, e4m3 (8) or e2m1 (4; two to a byte, the
 * even element in the low half), and stands for 2^(E - 127) code, exactly a bf16
 * (with E from 10 on, which is all that the append writes; of lower ones what is below
 * 2^-126 may count as 0).
 * kcache and vcache are blocks of bytes, shape.kv_stride BYTES apart (a multiple
 * of 16, at least mxfa_mx_block_bytes); in a block lie the codes [KV head][token]
 * [head_dim bits / 8], then the bytes E [KV head][token][head_dim / 32]. The other
 * fields of mxfa_batch_shape, and the tables, are as for the ordinary cache; dtype
 * is that of qkv, q and the outputs. The upkeep of pages is the ordinary one
 * (mxfa_run_pages_copy with a block of kv_stride bytes). */
/* The least bytes of a block, a multiple of 16; 0 where bits, head_dim (a multiple
 * of 32, at most 256) or block_size (a power of two) is not taken or they pass
 * an int. */
size_t mxfa_mx_block_bytes(int block_size, int n_kv_head, int head_dim, int bits);

/* As mxfa_run_cache_append, K and V quantised as they are written. E is the least,
 * 10 or more, by which the largest of the 32 is at most 448 2^(E - 127) (8 bits)
 * or 7 2^(E - 127) (4 bits: from 6 on it rounds to 6); the codes are the nearest,
 * on a tie the even one (elements above 1.75 2^127 count as that, whose code is in
 * the types' range). 32 elements of which one is not finite get E = 255 and
 * read back as NaN. K turns in 64 bits, rounded to 32, so equal tokens get equal
 * codes whatever computes them; factor is one of 64 bits for that. head_dim: a
 * multiple of 32, at most 256. The caches must not lie over each other, qkv or q_out
 * (MXFA_ERR_UNSUPPORTED); they may be columns of the same wider rows. */
typedef struct {
    int rotary_dim, interleaved;
    double factor;
    const double *frequencies; /* device, rotary_dim / 2 */
} mxfa_append_rotary_mx;
int mxfa_run_cache_append_mx(const mxfa_batch_shape *shape, int bits, const mxfa_append_rotary_mx *rotary,
                             const void *qkv, void *q_out, void *kcache, void *vcache, const int *block_table,
                             const int *cu_q, const int *lens, void *stream);

/* Rows back out of it: row r of k_out and v_out (n_tok rows, out_stride elements
 * apart, KV head h at elements [h head_dim, (h + 1) head_dim)) is what the cache
 * holds at the position of the append's row r for the same cu_q and lens: of each
 * sequence its last cu_q[s + 1] - cu_q[s] positions, all of them where that is
 * lens[s]. Rows at negative positions, past the table or in a block outside the
 * pool stay as they were. Reads neither n_head, q_stride nor scale. k_out and v_out
 * must not lie over each other or the caches (MXFA_ERR_UNSUPPORTED). */
int mxfa_run_cache_read_mx(const mxfa_batch_shape *shape, int bits, const void *kcache, const void *vcache, void *k_out,
                           void *v_out, const int *block_table, const int *cu_q, const int *lens, void *stream);

/* As mxfa_run_prefill_batch over what a microscaled cache holds. The workspace is
 * sized by mxfa_prefill_batch_mx_workspace_bytes. */
int mxfa_check_batch_mx(const mxfa_batch_shape *shape, int bits);
size_t mxfa_prefill_batch_mx_workspace_bytes(const mxfa_batch_shape *shape, int bits);
int mxfa_run_prefill_batch_mx(const mxfa_batch_shape *shape, int bits, const void *q, const void *kcache,
                              const void *vcache, void *out, float *lse, const int *block_table, const int *cu_q,
                              const int *lens, void *workspace, size_t workspace_bytes, void *stream);

/* ---- The pages of a cache: block tables (int32, table_stride elements between
 * rows), lengths and use counts of the blocks (int32 per block, how many table
 * rows hold it), all on the device. A sequence of lens[s] tokens holds its
 * row's first ceil(lens[s] / block_size) entries. */
typedef struct {
    int n_seq, max_blocks, table_stride, block_size, n_blocks;
} mxfa_pages_shape;
int mxfa_check_pages(const mxfa_pages_shape *shape);
/* The sequences rows[0 .. n - 1] end: the counts of their blocks go down, their
 * table entries become -1 and their lengths 0. Rows outside 0 .. n_seq - 1 are
 * skipped; a row named twice ends once. */
int mxfa_run_pages_free(const mxfa_pages_shape *shape, int *block_table, int *lens, int *refs, const int *rows, int n,
                        void *stream);
/* Row children[i] becomes a continuation of row parents[i]: it shares the
 * parent's whole blocks (their counts go up), and a last block that is not
 * full is to be copied to the lowest block that nobody uses (in the order of
 * the pairs). pairs[2j], pairs[2j + 1]: the j-th copy's source and destination
 * (n pairs of space); counts[0]: the copies, counts[1]: the refused pairs;
 * status[i]: 0, or 1 where the pair was refused and nothing done for it: a
 * row out of range, a child whose length is not 0, a child that an earlier
 * pair names, a parent longer than its row, or no block left. Parents count
 * as they were before the call. */
int mxfa_run_pages_fork(const mxfa_pages_shape *shape, int *block_table, int *lens, int *refs, const int *parents,
                        const int *children, int n, int *pairs, int *status, int *counts, void *stream);
/* The used blocks to the pool's low end: with L blocks in use, the j-th used
 * one at or above L moves to the j-th unused one below it. Writes the tables
 * and counts as they are after the moves (new_table may be block_table, with the
 * same stride, and else lies apart from it; new_refs lies apart from refs), the moves to pairs (n_blocks / 2 pairs of space,
 * at least one), and to counts how many and L. Until the blocks that were left
 * are used again, the old tables stay valid too. */
int mxfa_run_pages_compact(const mxfa_pages_shape *shape, const int *block_table, const int *lens, const int *refs,
                           int *new_table, int new_stride, int *new_refs, int *pairs, int *counts, void *stream);
/* Copies block pairs[2j] to block pairs[2j + 1], j < n_pairs (and < *count,
 * where count is not NULL: a device int), in each of n_pools pools pool_bytes
 * apart, of n_blocks blocks of block_bytes bytes. Pairs with a number outside
 * the pool are skipped. No destination may be another pair's source or
 * destination (not checked; the two calls above give none). */
int mxfa_run_pages_copy(void *pools, int n_pools, long long pool_bytes, int n_blocks, long long block_bytes,
                        const int *pairs, int n_pairs, const int *count, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MXFA_H */
