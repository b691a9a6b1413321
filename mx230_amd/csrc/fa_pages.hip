// Upkeep of a paged KV cache on the device: block tables, lengths and use
// counts of the pool's blocks, and the moves of their data.
//
// Bound: the copies by memory (2000 blocks of 16 rows x 2 KB in 8 pools: 213 us, 4.9
// TB/s, a large copy's rate); the rest by latency (tables of some thousand
// entries): one work-group plans what needs an order, so that equal inputs
// give equal blocks, and the rest is spread. us, 8 parents with 8 children of up to
// 4096 tokens: free 3.2, plan 5.7, rows 3.9, copies in 48 pools 5.4; the plan of a
// compaction of 8192 blocks 13.4, its tables 5.7.
#include <algorithm>

#include "fa_cache.h"
#include "fa_launch.h"

namespace mxfa {

constexpr int kPlan = 1024;  // threads of a planning work-group

// Blocks that hold a sequence of `len` tokens, within its table row.
__device__ __forceinline__ int row_blocks(const PagesParams &p, int len) {
    if (len <= 0) return 0;
    return min((int)(((long long)len + (1 << p.bs_shift) - 1) >> p.bs_shift), p.max_blocks);
}

// A value other threads of the work-group may have changed with an atomic (the
// L1 may hold the old one).
__device__ __forceinline__ int load_now(const int *x) {
    return __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_now(int *x, int v) {
    __hip_atomic_store(x, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive prefix of x over the kPlan threads, and the sum (in *total). Two
// barriers inside.
__device__ __forceinline__ int plan_prefix(int x, int *sums, int *total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlan / 64; ++w) {
        const int s = sums[w];
        before += w < wave ? s : 0;
        all += s;
    }
    *total = all;
    return before + inc - x;
}

// Sequence rows[i] ends: its blocks' counts go down, its row is emptied. The
// row's length is taken with an exchange, so a row named twice ends once.
__device__ __forceinline__ void pages_free_body(const PagesParams &p, const int *rows) {
    __shared__ int len;
    const int row = rows[blockIdx.x];
    if ((unsigned)row >= (unsigned)p.n_seq) return;
    if (threadIdx.x == 0) len = atomicExch(p.lens + row, 0);
    __syncthreads();
    int *t = p.table + (long long)row * p.table_stride;
    const int n = row_blocks(p, len);
    for (int j = threadIdx.x; j < n; j += 256) {
        const int b = t[j];
        t[j] = -1;
        if ((unsigned)b < (unsigned)p.n_blocks) atomicSub(p.refs + b, 1);
    }
}

// The fork's plan, one work-group: which pairs are taken (an empty child row,
// named for the first time, a parent that exists, a free block where the last
// one must be copied), the copies in the order of the pairs, from the lowest
// free blocks up, and the children's lengths and last blocks.
template <class Share>
__device__ __forceinline__ void pages_fork_plan(const PagesParams &p, const int *parents, const int *children, int m,
                                                int *pairs, int *status, int *counts, Share share) {
    __shared__ int sums[kPlan / 64];
    const int tid = threadIdx.x, part = (1 << p.bs_shift) - 1;
    // the parent's length where the pair may be taken, else -1
    for (int i = tid; i < m; i += kPlan) {
        const int a = parents[i], c = children[i];
        int len = -1;
        if ((unsigned)a < (unsigned)p.n_seq && (unsigned)c < (unsigned)p.n_seq && p.lens[c] == 0) {
            len = max(p.lens[a], 0);
            if (((long long)len + part) >> p.bs_shift > p.max_blocks) len = -1;
        }
        status[i] = len;
    }
    __syncthreads();
    // the first pair that names a child claims it
    for (int i = tid; i < m; i += kPlan) {
        if (status[i] >= 0) atomicMin(p.lens + children[i], i - m);
    }
    __syncthreads();
    int need = 0, refused = 0;  // the same in every thread
    for (int i0 = 0; i0 < m; i0 += kPlan) {
        const int i = i0 + tid;
        bool copy = false, no = false;
        if (i < m) {
            const int len = status[i], c = children[i];
            if (len < 0 || load_now(p.lens + c) != i - m) {
                status[i] = -1;
                no = true;
            } else {
                copy = (len & part) != 0;
            }
        }
        int total;  // (both counts in one, up to kPlan each)
        const int k = need + (plan_prefix(copy + (no << 16), sums, &total) & 0xffff);
        need += total & 0xffff;
        refused += total >> 16;
        // the copy's number, in the child's own row for now
        if (copy) p.table[(long long)children[i] * p.table_stride + (status[i] >> p.bs_shift)] = k;
    }
    // the lowest `need` blocks that nobody uses
    int found = 0;
    for (int b0 = 0; b0 < p.n_blocks && found < need; b0 += 4 * kPlan) {
        int free = 0, r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int b = b0 + 4 * tid + e;
            r[e] = b < p.n_blocks ? p.refs[b] : 1;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) free += r[e] == 0;
        int total, k = found + plan_prefix(free, sums, &total);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (r[e] == 0) {
                if (k < need) pairs[2 * k + 1] = b0 + 4 * tid + e;
                ++k;
            }
        }
        found += total;
    }
    found = min(found, need);
    __syncthreads();
    for (int i = tid; i < m; i += kPlan) {
        const int len = status[i];
        if (len < 0) {
            status[i] = 1;
            continue;
        }
        const int c = children[i];
        status[i] = 0;
        if (len & part) {
            int *last = p.table + (long long)c * p.table_stride + (len >> p.bs_shift);
            const int k = *last;
            if (k >= found) {  // no block left
                *last = -1;
                status[i] = 1;
                store_now(p.lens + c, 0);
                continue;
            }
            const int dst = pairs[2 * k + 1];
            pairs[2 * k] = p.table[(long long)parents[i] * p.table_stride + (len >> p.bs_shift)];
            *last = dst;
            p.refs[dst] = 1;
        }
        store_now(p.lens + c, len);
    }
    if (tid == 0) {
        counts[0] = found;
        counts[1] = refused + need - found;
    }
    __syncthreads();
    share();
}

// Entry j of pair i's rows: a whole block of the parent is shared.
__device__ __forceinline__ void pages_fork_entry(const PagesParams &p, const int *parents, const int *children,
                                                 const int *status, int i, int j) {
    if (status[i] != 0) return;
    const int c = children[i];
    if (j >= load_now(p.lens + c) >> p.bs_shift) return;
    const int b = p.table[(long long)parents[i] * p.table_stride + j];
    p.table[(long long)c * p.table_stride + j] = b;
    if ((unsigned)b < (unsigned)p.n_blocks) atomicAdd(p.refs + b, 1);
}

// The fork's rows where they are many, a work-group per pair.
__device__ __forceinline__ void pages_fork_rows(const PagesParams &p, const int *parents, const int *children,
                                                const int *status) {
    const int i = blockIdx.x;
    if (status[i] != 0) return;
    const int n = p.lens[children[i]] >> p.bs_shift;
    for (int j = threadIdx.x; j < n; j += 256) pages_fork_entry(p, parents, children, status, i, j);
}

// The compaction's plan, one work-group: with L used blocks in all, the j-th
// used block at or above L moves to the j-th unused one below it.
constexpr int kPlanEach = 8;  // consecutive blocks per thread and turn
__device__ __forceinline__ void pages_compact_plan(const PagesParams &p, int *new_refs, int *pairs, int *counts) {
    __shared__ int sums[kPlan / 64];
    const int tid = threadIdx.x;
    int r[kPlanEach], used = 0, live;
    auto read = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kPlanEach; ++e) {
            const int b = b0 + kPlanEach * tid + e;
            r[e] = b < p.n_blocks ? max(p.refs[b], 0) : 0;
        }
    };
    for (int b0 = 0; b0 < p.n_blocks; b0 += kPlanEach * kPlan) {
        read(b0);
#pragma unroll
        for (int e = 0; e < kPlanEach; ++e) used += r[e] > 0;
    }
    plan_prefix(used, sums, &live);
    int moved = 0, holes = 0;
    for (int b0 = 0; b0 < p.n_blocks; b0 += kPlanEach * kPlan) {
        if (p.n_blocks > kPlanEach * kPlan) read(b0);  // (else still there)
        int n = 0;  // moves, and holes from bit 16 on: up to kPlanEach kPlan each
#pragma unroll
        for (int e = 0; e < kPlanEach; ++e) {
            const int b = b0 + kPlanEach * tid + e;
            n += (b >= live && r[e] > 0) + ((b < live && r[e] == 0) << 16);
        }
        int total;
        const int k = plan_prefix(n, sums, &total);
        int km = moved + (k & 0xffff), kh = holes + (k >> 16);
#pragma unroll
        for (int e = 0; e < kPlanEach; ++e) {
            const int b = b0 + kPlanEach * tid + e;
            if (b < p.n_blocks) {
                if (b >= live && r[e] > 0) pairs[2 * km++] = b;
                if (b < live && r[e] == 0) pairs[2 * kh++ + 1] = b;
                new_refs[b] = b < live ? r[e] : 0;
            }
        }
        moved += total & 0xffff;
        holes += total >> 16;
    }
    __syncthreads();
    for (int j = tid; j < moved; j += kPlan) new_refs[pairs[2 * j + 1]] = p.refs[pairs[2 * j]];
    if (tid == 0) {
        counts[0] = moved;
        counts[1] = live;
    }
}

// The tables after the moves, a work-group per 256 entries: a moved block's
// number is found among the moves, which are in ascending order.
__device__ __forceinline__ void pages_compact_table(const PagesParams &p, int *new_table, int new_stride,
                                                    const int *pairs, const int *counts) {
    const int s = blockIdx.y, j = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (j >= p.max_blocks) return;
    int b = p.table[(long long)s * p.table_stride + j];
    const int moved = counts[0], live = counts[1];
    if (b >= live && j < row_blocks(p, p.lens[s])) {
        int lo = 0, hi = moved;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (pairs[2 * mid] < b) lo = mid + 1;
            else hi = mid;
        }
        if (lo < moved && pairs[2 * lo] == b) b = pairs[2 * lo + 1];
    }
    new_table[(long long)s * new_stride + j] = b;
}

// Whole blocks from pairs' first to their second, in every pool: a wave per
// 4 KB piece, in turns over the grid.
constexpr int kPiece = 4096;
__device__ __forceinline__ void pages_copy_body(char *pools, int n_pools, long long pool_bytes, int n_blocks,
                                                long long block_bytes, const int *pairs, int n_pairs,
                                                const int *count) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + ((int)threadIdx.x >> 6));
    const long long pieces = (block_bytes + kPiece - 1) / kPiece;
    const int n = count != nullptr ? min(max(*count, 0), n_pairs) : n_pairs;
    const long long all = pieces * n_pools * n;
    for (long long w = wave; w < all; w += (long long)gridDim.x * 4) {
        const long long pp = w / pieces, piece = w - pp * pieces;
        const int pool = (int)(pp % n_pools), i = (int)(pp / n_pools);
        const int src = pairs[2 * i], dst = pairs[2 * i + 1];
        if ((unsigned)src >= (unsigned)n_blocks || (unsigned)dst >= (unsigned)n_blocks || src == dst) continue;
        char *base = pools + pool * pool_bytes;
        const char *from = base + src * block_bytes + piece * kPiece;
        char *to = base + dst * block_bytes + piece * kPiece;
        const long long left = block_bytes - piece * kPiece;
        if (left >= kPiece) {
            const uint4 *f = reinterpret_cast<const uint4 *>(from) + lane;
            uint4 *t = reinterpret_cast<uint4 *>(to) + lane;
            const uint4 x0 = f[0], x1 = f[64], x2 = f[128], x3 = f[192];
            t[0] = x0;
            t[64] = x1;
            t[128] = x2;
            t[192] = x3;
        } else {
            for (long long o = lane * 16; o < left; o += 1024)
                *reinterpret_cast<uint4 *>(to + o) = *reinterpret_cast<const uint4 *>(from + o);
        }
    }
}

#if defined(__HIP_DEVICE_COMPILE__)
extern "C" __global__ __launch_bounds__(256) void mxfa_pages_free(PagesParams p, const int *rows) {
    pages_free_body(p, rows);
}
extern "C" __global__ __launch_bounds__(kPlan) void mxfa_pages_fork_plan(PagesParams p, const int *parents,
                                                                         const int *children, int m, int *pairs,
                                                                         int *status, int *counts, int rows) {
    pages_fork_plan(p, parents, children, m, pairs, status, counts, [&]() __attribute__((always_inline)) {
        for (int x = threadIdx.x; x < rows; x += kPlan) {
            const int i = x / p.max_blocks;
            pages_fork_entry(p, parents, children, status, i, x - i * p.max_blocks);
        }
    });
}
extern "C" __global__ __launch_bounds__(256) void mxfa_pages_fork_rows(PagesParams p, const int *parents,
                                                                       const int *children, const int *status) {
    pages_fork_rows(p, parents, children, status);
}
extern "C" __global__ __launch_bounds__(kPlan) void mxfa_pages_compact_plan(PagesParams p, int *new_refs, int *pairs,
                                                                            int *counts) {
    pages_compact_plan(p, new_refs, pairs, counts);
}
extern "C" __global__ __launch_bounds__(256) void mxfa_pages_compact_table(PagesParams p, int *new_table,
                                                                           int new_stride, const int *pairs,
                                                                           const int *counts) {
    pages_compact_table(p, new_table, new_stride, pairs, counts);
}
extern "C" __global__ __launch_bounds__(256) void mxfa_pages_copy(char *pools, int n_pools, long long pool_bytes,
                                                                  int n_blocks, long long block_bytes, const int *pairs,
                                                                  int n_pairs, const int *count) {
    pages_copy_body(pools, n_pools, pool_bytes, n_blocks, block_bytes, pairs, n_pairs, count);
}
#endif

hipError_t launch_pages_free(const PagesParams &p, const int *rows, int n, hipStream_t stream) {
    PagesParams q = p;
    void *args[] = {&q, &rows};
    return launch_kernel(k_mxfa_pages_free, dim3(n), dim3(256), args, stream);
}

// Entries of all pairs' rows up to which the plan's work-group shares the blocks
// itself instead of a second launch. us, rows ended and forked again: 4 pairs of 64
// blocks 9.0 (two launches 11.0), 8 of 256 11.7 (11.8), 16 of 256 14.5 (11.8).
constexpr int kForkOwn = 2048;
hipError_t launch_pages_fork(const PagesParams &p, const int *parents, const int *children, int n, int *pairs,
                             int *status, int *counts, hipStream_t stream) {
    PagesParams q = p;
    const long long entries = (long long)n * p.max_blocks;
    int own = entries <= kForkOwn ? (int)entries : 0;
    void *plan[] = {&q, &parents, &children, &n, &pairs, &status, &counts, &own};
    const hipError_t e = launch_kernel(k_mxfa_pages_fork_plan, dim3(1), dim3(kPlan), plan, stream);
    if (e != hipSuccess || entries == own) return e;
    void *rows[] = {&q, &parents, &children, &status};
    return launch_kernel(k_mxfa_pages_fork_rows, dim3(n), dim3(256), rows, stream);
}

hipError_t launch_pages_compact(const PagesParams &p, int *new_table, int new_stride, int *new_refs, int *pairs,
                                int *counts, hipStream_t stream) {
    PagesParams q = p;
    void *plan[] = {&q, &new_refs, &pairs, &counts};
    const hipError_t e = launch_kernel(k_mxfa_pages_compact_plan, dim3(1), dim3(kPlan), plan, stream);
    if (e != hipSuccess) return e;
    void *table[] = {&q, &new_table, &new_stride, &pairs, &counts};
    return launch_kernel(k_mxfa_pages_compact_table, dim3((p.max_blocks + 255) / 256, p.n_seq), dim3(256), table, stream);
}

hipError_t launch_pages_copy(void *pools, int n_pools, long long pool_bytes, int n_blocks, long long block_bytes,
                             const int *pairs, int n_pairs, const int *count, hipStream_t stream) {
    const double waves = (double)((block_bytes + kPiece - 1) / kPiece) * n_pools * n_pairs;
    // at most 8 work-groups of 4 waves on each of the 256 CUs
    const unsigned groups = (unsigned)std::min(2048.0, (waves + 3) / 4);
    void *args[] = {&pools, &n_pools, &pool_bytes, &n_blocks, &block_bytes, &pairs, &n_pairs, &count};
    return launch_kernel(k_mxfa_pages_copy, dim3(std::max(groups, 1u)), dim3(256), args, stream);
}

}  // namespace mxfa
