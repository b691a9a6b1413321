// The kernels of the gfx950 code object (mxfa_gfx950.hsaco), by name.
//
// This list is the one source of the names: the device sources define one
// `extern "C" __global__` kernel per entry (each an instantiation of a
// templated body), and the host library looks every entry up with
// hipModuleGetFunction when it loads the code object; a name missing from
// the code object fails that load. Naming: pass, dtype and head dim (b64 =
// bf16 d = 64, b128, f64 = fp32 d = 64), c / n = causal / not, then the
// variant (waves per SIMD w*, query tiles per wave q*, d = computes Delta,
// pg = K/V through a block table, g8 = 8 waves per work-group, few = at most 16 query rows, sp = one split of the keys, p2 = a softmax
// scale that is a power of two).
#pragma once

#define MXFA_KERNEL_LIST(X)                                                                   \
    /* forward (fa_fwd.hip): waves per SIMD, 16-query tiles per wave */                      \
    X(mxfa_fwd_b64_c_w3_q2) X(mxfa_fwd_b64_c_w3_q1)                                           \
    X(mxfa_fwd_b64_n_w2_q2) X(mxfa_fwd_b64_n_w3_q1)                                           \
    X(mxfa_fwd_b128_c_w2_q2) X(mxfa_fwd_b128_c_w2_q1) X(mxfa_fwd_b128_n_w2_q2)                \
    X(mxfa_fwd_f64_c) X(mxfa_fwd_f64_n) X(mxfa_fwd_f64_c_g8) X(mxfa_fwd_f64_n_g8)              \
    X(mxfa_fwd_b64_c_w3_q2_pg) X(mxfa_fwd_b64_c_w3_q1_pg)                                     \
    X(mxfa_fwd_b128_c_w2_q1_pg)                                                               \
    X(mxfa_fwd_f64_c_pg) X(mxfa_fwd_f64_c_pg_g8)                                              \
    X(mxfa_fwd_f64_c_sp_g8) X(mxfa_fwd_f64_c_pg_sp_g8)                                        \
    X(mxfa_fwd_b64_c_w3_q1_sp) X(mxfa_fwd_b128_c_w2_q1_sp) X(mxfa_fwd_f64_c_sp)                \
    X(mxfa_fwd_b64_c_w3_q1_pg_sp) X(mxfa_fwd_b128_c_w2_q1_pg_sp) X(mxfa_fwd_f64_c_pg_sp)       \
    X(mxfa_fwd_merge8_b64) X(mxfa_fwd_merge8_b128) X(mxfa_fwd_merge8_f64)                     \
    X(mxfa_fwd_merge32_b64) X(mxfa_fwd_merge32_b128) X(mxfa_fwd_merge32_f64)                  \
    X(mxfa_fwd_merge32t_b64) X(mxfa_fwd_merge32t_b128) X(mxfa_fwd_merge32t_f64)               \
    X(mxfa_fwd_merge128_b64) X(mxfa_fwd_merge128_b128)                                        \
    X(mxfa_fwd_b64_few) X(mxfa_fwd_b64_few_pg) X(mxfa_fwd_b64_few_sp) X(mxfa_fwd_b64_few_pg_sp) \
    X(mxfa_fwd_b128_few) X(mxfa_fwd_b128_few_pg) X(mxfa_fwd_b128_few_sp) X(mxfa_fwd_b128_few_pg_sp) \
    /* backward (fa_bwd.hip) */                                                               \
    X(mxfa_preprocess_b64) X(mxfa_preprocess_b128) X(mxfa_preprocess_f64)                     \
    X(mxfa_dq_b64_c) X(mxfa_dq_b64_c_d) X(mxfa_dq_b64_n) X(mxfa_dq_b64_n_d)                   \
    X(mxfa_dq_b128_c) X(mxfa_dq_b128_c_d) X(mxfa_dq_b128_n) X(mxfa_dq_b128_n_d)               \
    X(mxfa_dq_f64_c) X(mxfa_dq_f64_c_d) X(mxfa_dq_f64_n) X(mxfa_dq_f64_n_d)                   \
    X(mxfa_dkv_b64_c) X(mxfa_dkv_b64_n) X(mxfa_dkv_b128_c) X(mxfa_dkv_b128_n)                 \
    X(mxfa_bwd_f64_c) X(mxfa_bwd_f64_n)                                                       \
    X(mxfa_dkv_f64_c) X(mxfa_dkv_f64_n) X(mxfa_dkv_b64_c_p2) X(mxfa_dkv_b64_n_p2)             \
    X(mxfa_bwd_b64_c) X(mxfa_bwd_b64_n) X(mxfa_bwd_b128_c) X(mxfa_bwd_b128_n)                 \
    X(mxfa_bwd_b64_c_p2) X(mxfa_bwd_b64_n_p2)                                                 \
    X(mxfa_bwd_b64_c_w2) X(mxfa_bwd_b64_n_w2) X(mxfa_bwd_b64_c_p2_w2) X(mxfa_bwd_b64_n_p2_w2)  \
    X(mxfa_dkv_reduce_bf16) X(mxfa_dkv_reduce_f32)                                            \
    /* naive baselines (fa_naive.hip) */                                                      \
    X(mxfa_naive_scores) X(mxfa_naive_softmax) X(mxfa_naive_av) X(mxfa_naive_bwd)            \
    /* attention of a batch over a paged cache (fa_batch.hip) */                              \
    X(mxfa_batch_b64_few) X(mxfa_batch_b64_many) X(mxfa_batch_b64_join) X(mxfa_batch_b64_both)                       \
    X(mxfa_batch_b128_few) X(mxfa_batch_b128_many) X(mxfa_batch_b128_join) X(mxfa_batch_b128_both)                    \
    X(mxfa_batch_b64_many64) X(mxfa_batch_b64_both64) X(mxfa_batch_b128_many64) X(mxfa_batch_b128_both64)             \
    X(mxfa_batch_f64_few) X(mxfa_batch_f64_many) X(mxfa_batch_f64_join) X(mxfa_batch_f64_both)                       \
    /* attention of a batch over a microscaled cache (fa_batch_mx.hip): x8 or x4, then the type and head dim */ \
    X(mxfa_batch_x8b64_few) X(mxfa_batch_x8b64_one) X(mxfa_batch_x8b64_many) X(mxfa_batch_x8b64_both) X(mxfa_batch_x8b64_many64) X(mxfa_batch_x8b64_both64) \
    X(mxfa_batch_x8b128_few) X(mxfa_batch_x8b128_one) X(mxfa_batch_x8b128_many) X(mxfa_batch_x8b128_both) X(mxfa_batch_x8b128_many64) X(mxfa_batch_x8b128_both64) \
    X(mxfa_batch_x8f64_few) X(mxfa_batch_x8f64_one) X(mxfa_batch_x8f64_many) X(mxfa_batch_x8f64_both) \
    X(mxfa_batch_x4b64_few) X(mxfa_batch_x4b64_one) X(mxfa_batch_x4b64_many) X(mxfa_batch_x4b64_both) X(mxfa_batch_x4b64_many64) X(mxfa_batch_x4b64_both64) \
    X(mxfa_batch_x4b128_few) X(mxfa_batch_x4b128_one) X(mxfa_batch_x4b128_many) X(mxfa_batch_x4b128_both) X(mxfa_batch_x4b128_many64) X(mxfa_batch_x4b128_both64) \
    X(mxfa_batch_x4f64_few) X(mxfa_batch_x4f64_one) X(mxfa_batch_x4f64_many) X(mxfa_batch_x4f64_both) \
    /* its append and its read (fa_mx.hip) */ \
    X(mxfa_append_x8b) X(mxfa_append_x8b1) X(mxfa_append_x8f) X(mxfa_append_x8f1) X(mxfa_read_x8b) X(mxfa_read_x8f) \
    X(mxfa_append_x4b) X(mxfa_append_x4b1) X(mxfa_append_x4f) X(mxfa_append_x4f1) X(mxfa_read_x4b) X(mxfa_read_x4f) \
    /* rotary positions and the cache append (fa_rotary.hip): 16-byte, 8-byte, single-element chunks */ \
    X(mxfa_rotary_b) X(mxfa_rotary_b4) X(mxfa_rotary_b1) X(mxfa_rotary_f) X(mxfa_rotary_f1)   \
    X(mxfa_append_b) X(mxfa_append_b4) X(mxfa_append_b1) X(mxfa_append_f) X(mxfa_append_f1)   \
    /* the pages of a cache (fa_pages.hip) */                                                 \
    X(mxfa_pages_free) X(mxfa_pages_fork_plan) X(mxfa_pages_fork_rows)                        \
    X(mxfa_pages_compact_plan) X(mxfa_pages_compact_table) X(mxfa_pages_copy)                 \
    /* probes (probe.hip) */                                                                  \
    X(mxfa_probe_mfma_bf16) X(mxfa_probe_mfma_f32) X(mxfa_probe_mfma32_bf16)                  \
    X(mxfa_probe_read_f4) X(mxfa_probe_copy_f4) X(mxfa_probe_dq_atomic_add)                   \
    X(mxfa_probe_dq_atomic_store) X(mxfa_probe_mix_mfma) X(mxfa_probe_mix_dkv)                  \
    X(mxfa_probe_mix_dkv_valu) X(mxfa_probe_mix_dkv_lds) X(mxfa_probe_mix_dq) X(mxfa_probe_mix_fwd)         \
    X(mxfa_probe_mix32_mfma) X(mxfa_probe_mix32_dkv) X(mxfa_probe_mix32_dq) X(mxfa_probe_mix32_fwd)

namespace mxfa {

enum KernelId {
#define MXFA_KID(n) k_##n,
    MXFA_KERNEL_LIST(MXFA_KID)
#undef MXFA_KID
    kNumKernels
};

}  // namespace mxfa
