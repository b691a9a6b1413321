// Parameters and launchers of the operators around the attention kernels:
// rotary positions, the cache append, attention of a batch over a paged cache
// and the upkeep of its pages (internal to libmxfa; shapes are validated by
// the C ABI, mxfa_api.cpp, before any launcher is called).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mxfa {

// One tensor of heads: strides in elements between batches, heads and tokens.
struct HeadView {
    const void *in;
    void *out;
    long long in_bs, in_hs, in_ts, out_bs, out_hs, out_ts;
};

struct RotaryParams {
    HeadView x[2];  // Q and K (H[1] = 0: Q alone)
    int H[2];
    int B, N, d, dim, interleaved;
    int pos0;              // positions null: token n at pos0 + n
    const int *positions;  // else token n of batch b at positions[b pos_bs + n]
    long long pos_bs;
    const double *freq;    // dim / 2 angles per position, radians
    float factor, sin_sign;
    int hpt;  // heads per thread
};

// A batch of sequences whose new tokens are consecutive rows: sequence s has
// rows cu_q[s] .. cu_q[s + 1] - 1, the last of its lens[s] positions, and its
// cache rows through table[s table_stride + position / block size].
struct BatchParams {
    const void *q;
    void *k, *v, *o;
    float *lse;
    const int *table, *cu_q, *lens;
    int n_tok, n_seq, max_q, Hq, Hkv, group, d;
    int q_rs, kv_rs, o_rs, bs_shift, n_blocks, max_blocks, table_stride;
    float scale_log2;
    // append: the rotation of Q and K (dim = 0: none)
    const double *freq;
    int dim, interleaved;
    float factor;
    int hpt;  // heads per thread
    // attention (fa_batch_items.h): the most rows (new tokens x query heads of a
    // KV head) of a sequence that the few-row form takes (0: it takes none) and
    // its work-groups per KV head; the rows of the many-row form's
    // units; per form the least stages of a run or share; of the many-row form: what a split costs, in stages and in stages
    // per item (batch_quota), the work-groups resident at once, 1 / that, whether a
    // launch has more than those, the slots of its shares and the split units there can be; the forms' parts of the
    // workspace and their notes
    int few_rows, few_groups, many_rows, least[2], whole, resident, roomy, slots, splits;
    float per_item, per_resident;
    float *part[2];
    int *notes[2];
};

struct PagesParams {
    int *table, *lens, *refs;
    int n_seq, max_blocks, table_stride, bs_shift, n_blocks;
};

// The threads that a head's row takes (head dim d, `dim` of it rotated).
int rotary_row_units(int d, int dim, int dtype_bf16);
hipError_t launch_rotary(RotaryParams p, int dtype_bf16, hipStream_t stream);
hipError_t launch_append(BatchParams p, int dtype_bf16, hipStream_t stream);

// Attention of the batch's new tokens over the cache; p.part from a workspace of
// batch_workspace_bytes (set by the launcher).
size_t batch_workspace_bytes(const BatchParams &p, int dtype_bf16);
long long batch_groups(const BatchParams &p, int dtype_bf16);  // of the largest launch
hipError_t launch_batch(BatchParams p, int dtype_bf16, void *workspace, hipStream_t stream);

hipError_t launch_pages_free(const PagesParams &p, const int *rows, int n, hipStream_t stream);
hipError_t launch_pages_fork(const PagesParams &p, const int *parents, const int *children, int n, int *pairs,
                             int *status, int *counts, hipStream_t stream);
hipError_t launch_pages_compact(const PagesParams &p, int *new_table, int new_stride, int *new_refs, int *pairs,
                                int *counts, hipStream_t stream);
hipError_t launch_pages_copy(void *pools, int n_pools, long long pool_bytes, int n_blocks, long long block_bytes,
                             const int *pairs, int n_pairs, const int *count, hipStream_t stream);

}  // namespace mxfa
