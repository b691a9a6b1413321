// Attention of a batch of sequences' new tokens over a paged KV cache: each
// sequence has its own number of new tokens (one, or a chunk), its own length
// and its own row of the block table, all on the device.
//
//     o_i = sum_{j <= pos_i} p_ij v_j / sum_j p_ij,   p_ij = 2^(s_ij - m_i),
//     s_ij = q_i . k_j scale log2(e),                 lse_i = (m_i + log2 sum_j p_ij) ln 2,
//
// one pass over the keys with the running maximum m and sum. A sequence's rows
// of one KV head are its new tokens times the head's query heads (row r: token
// r / group, query head r % group), so that a key that is read serves the whole
// group. Sums, maxima and O are fp32; in bf16 p is rounded to bf16 for the product
// with V (relative 2^-8 at most, each p by itself), as the matrix instruction takes
// it, and its sum is of the values before that. fp32 operands keep 24 bits.
//
// Two forms take a sequence's rows in units:
//   * few (at most 16 rows, one unit): every wave holds the same rows and takes
//     64-key stages of its own; bound by the reads of K and V;
//   * many: units of 128 or (bf16) 64 rows, the waves sharing each stage; bound by
//     the matrix products.
// The host knows neither lengths nor units, only the buffers' sizes: a work-group
// finds its part of the work from cu_q and lens itself (fa_batch_items.h has the
// arithmetic). Where a sequence's or unit's keys are several work-groups', their
// unnormalised outputs are joined by a second launch, in a fixed order, so equal
// calls give equal bits. A counter per unit would save that launch (4 to 7 us), but
// has to be cleared before each call, and an only reader per unit of up to 128
// parts takes longer than the many of the launch.
//
// Measured (us, medians of a kernel trace; the rates count the keys each sequence
// has once, or the products of the positions that rows see):
//   few:  64 sequences of one token, 2000-16384 long, 32/8 heads, d = 128: 391 and
//         the join 6 (2.2 GB, 5.6 TB/s; a plain read of all memory reaches 6.4), d =
//         64 221 and 6 (5.0), fp32 (d = 64) 414 and 7 (5.3);
//         one token after 4095, 32/4 heads, d = 64: 7.1 and 4.0, fp32 8.8 and 4.1;
//   many: the last 2048 tokens of 32768, 32/8 heads, d = 128: 920 to 970 in runs of
//         calls on different cards (1100 to 1150 TFLOP/s; a large library product
//         1180); 4096 tokens, 32/4 heads, d = 64: 87 to 90 (770); fp32, 2000 tokens
//         after 2096, 14/2 heads: 169 to 180 with the join (123 to 131; in fp32 150);
//   both: 28 single tokens and 4 chunks of up to 512, to 8192 long, 14/2 heads,
//         d = 64: 48.6 and the join 7 (one after the other: 41 and 18); 32/8 heads, d
//         = 128: 213 with the join (98.7 GFLOP, 0.65 GB); fp32, 6 tokens and 2 chunks
//         of up to 500, to 4096 long, 14/2 heads: 55 and 7.
#include <algorithm>
#include <type_traits>

#include "fa_batch_items.h"
#include "fa_device.h"
#include "fa_launch.h"

namespace mxfa {

// The device code builds on the forward's stages (fa_fwd.hip, the same
// translation unit in the code object).
#if defined(__HIP_DEVICE_COMPILE__)

// ------------------------------------------------- fp32 on its own instructions

// fp32 inputs (d = 64) on v_mfma_f32_16x16x4_f32, in the policy form of
// fwd_stage, for the few-row form, which the reads bound. LDS rows of 256 bytes
// hold their 16-byte chunk c at c ^ (row & 15), so the 16 rows of a score operand and the 16 chunks of a V row both cover
// all banks. Score k-steps: MFMA (c, e) takes element 16c + 4g + e of lane
// group g. In the chained product a lane reads 4 columns of a V row at once, so
// tile xt's row 4g + r of O^T is column 4 (4g + r) + xt.
struct PolF32 {
    static constexpr int D = 64;
    using T = float;
    using Frag = f32x4;
    static constexpr int EPC = 4, NC = 4, ROWS = 64;
    __device__ static __forceinline__ void chunk_at(int P, int &row, int &chunk) {
        row = P >> 4;
        chunk = (P & 15) ^ (row & 15);
    }
    __device__ static __forceinline__ constexpr int arow(int t, int m) { return 16 * t + m; }
    __device__ static __forceinline__ constexpr int bidx(int t, int g, int r) { return 16 * t + 4 * g + r; }
    __device__ static __forceinline__ int chunk_off(int row, int chunk) { return row * 256 + ((chunk ^ (row & 15)) << 4); }
    __device__ static __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    __device__ static __forceinline__ void lds_row_frags(Frag (&f)[NC], const T *tile, int n, int g) {
        const char *base = reinterpret_cast<const char *>(tile);
#pragma unroll
        for (int c = 0; c < NC; ++c) f[c] = *reinterpret_cast<const Frag *>(base + chunk_off(n, 4 * c + g));
    }
    struct ChainB {
        f32x4 c[2];
    };
    __device__ static __forceinline__ ChainB pack(const f32x4 &c0, const f32x4 &c1) { return ChainB{{c0, c1}}; }
    __device__ static __forceinline__ f32x4 chain(f32x4 acc, const ChainB &b, const T *tile, int y0, int blk, int g,
                                                  int l16) {
        const char *base = reinterpret_cast<const char *>(tile);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const Frag v = *reinterpret_cast<const Frag *>(base + chunk_off(blk + bidx(t, g, r), l16));
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v[y0 / 16], b.c[t][r], acc, 0, 0, 0);
            }
        }
        return acc;
    }
};

// bf16 inputs on v_mfma_f32_16x16x32_bf16 as PolBF16, from LDS tiles whose
// rows lie whole, one after another, so that a wave's staging load reads whole
// rows of the cache (4 rows of 256 bytes or 8 of 128; PolBF16's column groups
// take 32 bytes of each of 32 rows). Chunk c of row r (bits r0, r1, ...) is at
// slot c ^ swz(r). The 16 rows of a score operand differ in r0, r1, r3, r4, a
// transposing read of V takes two neighbouring chunks of rows differing in r0
// and r1 (two lane groups: r3), and the bit patterns below are to spread each of
// these over the banks, in 128- and in 256-byte halves. r2 and r5 (tile t or half h,
// block) stay out of it: plain additions. The counters still show conflicts in 31%
// of the LDS-active cycles of the many-row form, 25% of the few-row form's (PolBF16's
// tiles have none).
template <int D_>
struct PolRows {
    using Base = PolBF16<D_>;
    static constexpr int D = D_, EPC = 8, NC = Base::NC, ROWS = 64, CPR = D / 8;
    using T = u16;
    using Frag = typename Base::Frag;
    using ChainB = typename Base::ChainB;
    __device__ static __forceinline__ int arow(int t, int m) { return Base::arow(t, m); }
    __device__ static __forceinline__ int bidx(int t, int g, int r) { return Base::bidx(t, g, r); }
    __device__ static __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) { return Base::mma(a, b, c); }
    __device__ static __forceinline__ ChainB pack(const f32x4 &a, const f32x4 &b) { return Base::pack(a, b); }
    __device__ static __forceinline__ int swz(int r) {
        const int r0 = r & 1, r1 = (r >> 1) & 1, r3 = (r >> 3) & 1, r4 = (r >> 4) & 1;
        return D == 128 ? (2 * r0) ^ (4 * r1) ^ (9 * r3) ^ r4 : (5 * r0) ^ (2 * r1) ^ (4 * r3) ^ r4;
    }
    __device__ static __forceinline__ void lds_row_frags(Frag (&f)[NC], const T *tile, int n, int g) {
        const char *base = reinterpret_cast<const char *>(tile) + n * (2 * D);
        const int x = (g ^ swz(n)) << 4;
#pragma unroll
        for (int c = 0; c < NC; ++c) f[c] = *reinterpret_cast<const Frag *>(base + (x ^ (64 * c)));
    }
    __device__ static __forceinline__ f32x4 chain(f32x4 acc, const ChainB &b, const T *tile, int y0, int blk, int g,
                                                  int l16) {
        const int r0 = blk + 8 * g + (l16 >> 2);
        const char *base = reinterpret_cast<const char *>(tile) + r0 * (2 * D) + ((l16 & 1) << 3);
        const int x = (((l16 >> 1) & 1) ^ swz(r0)) << 4;
        const int off = x ^ (2 * y0);
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(base + off));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(base + off + 4 * (2 * D)));
        return mma(__builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), b, acc);
    }
    // the chunk at 16-byte position P of the tile, and its row
    __device__ static __forceinline__ void chunk_at(int P, int &row, int &chunk) {
        row = P / CPR;
        chunk = (P % CPR) ^ swz(row);
    }
};

// A row's elements that a lane holds as operand B of the scores.
template <class Pol>
__device__ __forceinline__ void row_frags(typename Pol::Frag (&f)[Pol::NC], const typename Pol::T *row, int g) {
    constexpr int S = sizeof(typename Pol::T) == 2 ? 8 : 4;
#pragma unroll
    for (int c = 0; c < Pol::NC; ++c) f[c] = *reinterpret_cast<const typename Pol::Frag *>(row + 4 * S * c + S * g);
}

// ------------------------------------------------------------- staging of pages

// Cache row of position t of a sequence whose block is `blk`, as an index: blocks
// outside the pool count as the nearest in it, so no read leaves the caches.
struct BatchRows {
    const int *table;
    int shift, keys;
    unsigned last;
    __device__ __forceinline__ int block_at(int t) const { return min(t, keys - 1) >> shift; }
    __device__ __forceinline__ unsigned row(int blk, int t) const {
        const unsigned off = (unsigned)min(t, keys - 1) & ((1u << shift) - 1u);
        return (min((unsigned)blk, last) << shift) + off;
    }
};

// The loads of one 64-key tile by NT threads: load k fills 16-byte positions k NT
// + tid, whole rows of the cache; off holds the loads' byte offsets in the cache
// (row_of(r): the cache row of the tile's row r). Rows may be more than 4 GiB
// apart: a stride of INT_MAX elements in bytes fits 32 bits in bf16 (one 32 x 32 bit
// product per load; with the shift of a product of elements instead 0.7% of
// 960 us, 2048 tokens of 32768, d = 128), in fp32 it takes 64.
template <class Pol, int NT>
struct BatchStage {
    static constexpr int CPR = Pol::D / Pol::EPC, LOADS = 64 * CPR / NT;
    using Stride = std::conditional_t<sizeof(typename Pol::T) == 2, unsigned, unsigned long long>;
    unsigned long long off[LOADS];
    __device__ static __forceinline__ Stride stride_bytes(int stride) { return (Stride)stride * (Stride)sizeof(typename Pol::T); }
    template <class RowOf>
    __device__ __forceinline__ void rows(int tid, Stride stride, RowOf row_of) {
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            int row, c;
            Pol::chunk_at(k * NT + tid, row, c);
            off[k] = (unsigned long long)row_of(row) * stride + 16 * c;
        }
    }
    __device__ __forceinline__ void load(typename Pol::T *tile, const typename Pol::T *X, int wave) const {
        const uint32_t base = lds_addr(tile) + wave * 64 * 16;
#pragma unroll
        for (int k = 0; k < LOADS; ++k) lds_dma16(base + k * NT * 16, reinterpret_cast<const char *>(X) + off[k]);
    }
};

// -------------------------------------------------------------------- the items

// Inclusive prefix over the wave, all 64 lanes active (rows of 16 by shifts, then
// the rows' ends broadcast into the next row, and into the upper half).
template <class X>
__device__ __forceinline__ X wave_prefix(X x) {
    auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                  decltype(rows)::value, 0xf, false);
        x += __builtin_bit_cast(X, o);
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast 15, 31
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
    return x;
}
template <class X>
__device__ __forceinline__ X wave_sum(X x) {
    return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_prefix(x)), 63));
}

__device__ __forceinline__ BatchSeq seq_of_lane(const BatchSeq &b, int l) {
    auto of = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
    return BatchSeq{of(b.q0), of(b.pos), of(b.rows), of(b.keys), of(b.units), of(b.stages)};
}

// Item `w` of the many-row form, found by every wave for itself: a lane per
// sequence, again over them where there are more than 64 (the rules:
// fa_batch_items.h). False past the last one. The work-group of item 0 also
// notes the count of split units for the join.
template <int ROWS>
__device__ __forceinline__ bool find_item(const BatchParams &p, int w, BatchItem &it) {
    const int lane = threadIdx.x & 63;
    BatchSeq b = batch_seq<false, ROWS>(p, lane);
    float all = seq_stages<ROWS>(p, b), units = (float)b.units;
    for (int s0 = 64; s0 < p.n_seq; s0 += 64) {
        const BatchSeq c = batch_seq<false, ROWS>(p, s0 + lane);
        all += seq_stages<ROWS>(p, c);
        units += (float)c.units;
    }
    auto count = [&](unsigned q) __attribute__((always_inline)) {
        int n = seq_items<ROWS>(p, b, q).items;
        for (int s0 = 64; s0 < p.n_seq; s0 += 64) n += seq_items<ROWS>(p, batch_seq<false, ROWS>(p, s0 + lane), q).items;
        return (float)wave_sum(n);
    };
    auto longer = [&](unsigned x) __attribute__((always_inline)) {
        bool is = (unsigned)b.stages > x;
        for (int s0 = 64; s0 < p.n_seq; s0 += 64) is |= (unsigned)batch_seq<false, ROWS>(p, s0 + lane).stages > x;
        return __builtin_amdgcn_ballot_w64(is) != 0;
    };
    const unsigned quota = batch_quota(p, wave_sum(all), wave_sum(units), count, longer);
    if (w == 0 && p.splits > 0) {
        int n = seq_items<ROWS>(p, b, quota).split;
        for (int s0 = 64; s0 < p.n_seq; s0 += 64) n += seq_items<ROWS>(p, batch_seq<false, ROWS>(p, s0 + lane), quota).split;
        n = wave_sum(n);
        if (threadIdx.x == 0) p.notes[1][0] = n;
    }
    int before = 0, slots = 0, splits = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        if (s0 > 0) b = batch_seq<false, ROWS>(p, s0 + lane);
        const SeqItems n = seq_items<ROWS>(p, b, quota);
        const int upto = wave_prefix(n.items), slots_upto = wave_prefix(n.slots), splits_upto = wave_prefix(n.split);
        const unsigned long long at = __builtin_amdgcn_ballot_w64(before + upto > w);
        if (at != 0) {
            const int l = __builtin_ctzll(at);
            auto of = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
            it.seq = s0 + l;
            it.s = seq_of_lane(b, l);
            const SeqItems m{of(n.whole), of(n.shares), of(n.split), of(n.slots), of(n.items)};
            if (!batch_item(p, m, slots + of(slots_upto - n.slots), splits + of(splits_upto - n.split),
                            w - before - of(upto - n.items), it))
                return false;
            if (it.shares > 1 && it.share == 0 && it.split < p.splits && threadIdx.x == 0)
                reinterpret_cast<ManyNote *>(p.notes[1])[1 + it.split] =
                    ManyNote{it.shares, it.slot, it.s.q0, it.s.rows, it.unit, it.head, {it.s.pos, 0}};
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slots_upto, 63);
        splits += __builtin_amdgcn_readlane(splits_upto, 63);
    }
    return false;
}

// The length of the few-row form's line.
__device__ __forceinline__ unsigned few_line(const BatchParams &p) {
    unsigned all = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) all += few_weight(batch_seq<true, kBatchFew>(p, s0 + (threadIdx.x & 63)));
    return wave_sum(all);
}

// f(sequence's number, BatchSeq, its begin and end on the line) for the sequences
// from position x of the line on, until f returns true.
template <class F>
__device__ __forceinline__ void few_walk(const BatchParams &p, unsigned x, F f) {
    const int lane = threadIdx.x & 63;
    unsigned before = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const BatchSeq b = batch_seq<true, kBatchFew>(p, s0 + lane);
        const unsigned w = few_weight(b), upto = before + wave_prefix(w);
        unsigned long long left = __builtin_amdgcn_ballot_w64(w > 0 && upto > x);
        for (; left != 0; left &= left - 1) {
            const int l = __builtin_ctzll(left);
            const unsigned u1 = __builtin_amdgcn_readlane(upto, l);
            if (f(s0 + l, seq_of_lane(b, l), u1 - __builtin_amdgcn_readlane(w, l), u1)) return;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
}

// Row r of a unit's sequence: its elements in q or o, and its index in lse.
__device__ __forceinline__ size_t batch_elem(const BatchParams &p, const BatchItem &it, int r, int stride, int d) {
    return (size_t)(it.s.q0 + r / p.group) * (size_t)stride + (size_t)(it.head * p.group + r % p.group) * d;
}
__device__ __forceinline__ size_t batch_lse(const BatchParams &p, const BatchItem &it, int r) {
    return (size_t)(it.s.q0 + r / p.group) * p.Hq + it.head * p.group + r % p.group;
}

// What the sum of V of a row at position `pos` is multiplied by, l being the sum
// of its weights: 0 where it sees no position; where every score that it sees is
// -infinity (K infinite, or products past the range) there is no softmax: NaN.
__device__ __forceinline__ float batch_inverse(float l, int pos) { return l != 0.f ? 1.0f / l : pos < 0 ? 0.f : NAN; }

// Four elements of a finished row, and its lse by the row's first thread.
template <class T>
__device__ __forceinline__ void batch_store(const BatchParams &p, const BatchItem &it, int r, int d, int c, f32x4 o,
                                            float m, float l) {
    T *O = static_cast<T *>(p.o) + batch_elem(p, it, r, p.o_rs, d) + c;
    store4<T>(O, o, batch_inverse(l, it.s.pos + r / p.group));
    if (p.lse != nullptr && c == 0) p.lse[batch_lse(p, it, r)] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

// The columns a lane holds of its row: 4 of them from batch_col(i, g), i < XT.
template <class Pol>
__device__ __forceinline__ int batch_col(int i, int g) {
    return sizeof(typename Pol::T) == 2 ? 16 * i + 4 * g : 16 * g + 4 * i;
}
template <class Pol, int XT, int QT>
__device__ __forceinline__ f32x4 batch_quad(const f32x4 (&acc)[XT][QT], int i, int qt) {
    if constexpr (sizeof(typename Pol::T) == 2) {
        return acc[i][qt];
    } else {
        return f32x4{acc[0][qt][i], acc[1][qt][i], acc[2][qt][i], acc[3][qt][i]};
    }
}

// A unit's share in plain fp32 arithmetic, keys a row does not see left out
// altogether: taken where a value was not finite, since in the matrix products
// an infinity or NaN in the V of a key that a row does not see reaches it as 0
// x inf. 4 threads per row, rows from row0 of the unit. Some 6 times the time of the
// products. A row's running (max, sum) and output go where the form's would: to the workspace slot, or (part null) finished.
template <class T, int D, int ROWS>
__device__ __forceinline__ void batch_plain(const BatchParams &p, const BatchItem &it, int row0, int key0, int key1,
                                            float *part, float *ml) {
    constexpr int E = D / 4;
    const int rl = (int)(threadIdx.x >> 2) + row0, c = E * (int)(threadIdx.x & 3);
    const int r = it.unit * ROWS + rl;
    const bool have = r < it.s.rows;
    const int row = min(r, it.s.rows - 1);
    const T *Q = static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D) + c;
    auto val = [](T x) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 2) return __uint_as_float((uint32_t)x << 16);
        else return x;
    };
    float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = val(Q[e]) * p.scale_log2;
        acc[e] = 0.f;
    }
    const int kend = min(min(key1, it.s.keys), it.s.pos + row / p.group + 1);
    const int *table = p.table + (long long)it.seq * p.table_stride;
    for (int k = key0; k < kend; ++k) {
        const size_t b = min((unsigned)table[k >> p.bs_shift], (unsigned)(p.n_blocks - 1));
        const size_t at = ((b << p.bs_shift) + (k & ((1 << p.bs_shift) - 1))) * (size_t)p.kv_rs + it.head * D + c;
        const T *K = static_cast<const T *>(p.k) + at, *V = static_cast<const T *>(p.v) + at;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = __builtin_fmaf(q[e], val(K[e]), s);
        s = quad_sum(s);
        const float mn = fmaxf(m, s), mref = mn == -INFINITY ? 0.f : mn;
        const float corr = fast_exp2(m - mref), pv = fast_exp2(s - mref);
        m = mn;
        l = l * corr + pv;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(pv, val(V[e]), acc[e] * corr);
    }
    if (!have) return;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const f32x4 o{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
        if (part != nullptr) {
            store4<float>(part + (size_t)rl * D + c + e, o, 1.0f);
        } else {
            batch_store<T>(p, it, r, D, c + e, o, m, l);
        }
    }
    if (part != nullptr && c == 0) *reinterpret_cast<float2 *>(ml + 2 * rl) = make_float2(m, l);
}

// A slot of a form's workspace: its units' rows of d floats, and their (max, sum).
__device__ __forceinline__ float *batch_part(float *part, int slot, int rows, int d) {
    return part + (size_t)slot * rows * d;
}
__device__ __forceinline__ float *batch_ml(float *part, int slots, int slot, int rows, int d) {
    return part + (size_t)slots * rows * d + (size_t)slot * rows * 2;
}
__device__ __forceinline__ int few_slots(const BatchParams &p) { return 2 * p.few_groups * p.Hkv; }

// ------------------------------------------------------------------ the few rows

template <class Pol, int NW>
union BatchFewSmem {
    struct {
        typename Pol::T k[NW][Pol::ROWS * Pol::D], v[NW][Pol::ROWS * Pol::D];
        int blk[NW][2][64];
    } t;
    struct {
        float acc[NW][kBatchFew][Pol::D + 4];
        float ml[NW][kBatchFew][2];
        int bad;
    } merge;
};

// One piece of a sequence: each of the NW waves takes every NW-th of its stages
// [s_lo, s_hi), staged into its own tiles with no barrier; the waves' maxima,
// sums and O meet in LDS. The stage's blocks come through LDS too, two stages
// ahead: as loads into registers the compiler would wait for them with
// vmcnt(0), and with them for every staging load in flight.
//
// Bound by the reads: 128 KB of tiles in flight per CU (8 waves of 16 KB, d = 128: 4
// of 32), and nothing but the next tile's loads between two waits. us, 64 sequences
// of 2000-16384 positions, 32/8 heads, d = 128, at the step that brought it: 411
// where a load reads whole rows, 510 by 32 bytes of each of 32 rows.
template <class Pol, int NW, int THREADS>
__device__ __forceinline__ void batch_few_piece(const BatchParams &p, const BatchItem &it, int s_lo, int s_hi, int slot,
                                                BatchFewSmem<Pol, NW> &sm) {
    using T = typename Pol::T;
    using Stage = BatchStage<Pol, 64>;
    constexpr int D = Pol::D, XT = D / 16, ROWS = kBatchFew, NL = Stage::LOADS;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const T *K = static_cast<const T *>(p.k) + it.head * D, *V = static_cast<const T *>(p.v) + it.head * D;
    const BatchRows rows{p.table + (long long)it.seq * p.table_stride, p.bs_shift, it.s.keys, (unsigned)(p.n_blocks - 1)};
    const typename Stage::Stride stride = Stage::stride_bytes(p.kv_rs);
    // waves past the NW that have tiles only take part in the join
    const int own = NW * 64 < THREADS ? min(wave, NW - 1) : wave;
    T *sk = sm.t.k[own], *sv = sm.t.v[own];
    const int Nk = it.s.keys;

    // stage `st` is the wave's n-th: its blocks in buffer n & 1
    auto fetch = [&](int st, int n) __attribute__((always_inline)) {
        lds_dma4(lds_addr(sm.t.blk[own][n & 1]), rows.table + rows.block_at(st * 64 + lane));
    };
    auto load = [&](T *tile, const T *X, int st, int n) __attribute__((always_inline)) {
        const int *blk = sm.t.blk[own][n & 1];
        Stage stage;
        stage.rows(lane, stride, [&](int r) __attribute__((always_inline)) { return rows.row(blk[r], st * 64 + r); });
        stage.load(tile, X, 0);
    };
    int st = wave < NW ? s_lo + wave : s_hi, n = 0;
    if (st < s_hi) fetch(st, 0);
    const int row = min(l16, it.s.rows - 1);
    const int qpos = it.s.pos + row / p.group;
    typename Pol::Frag qf[1][Pol::NC];
    row_frags<Pol>(qf[0], static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D), g);
    if (st < s_hi) {
        wait_loads<0>();
        if (st + NW < s_hi) fetch(st + NW, 1);
        load(sk, K, st, 0);
        load(sv, V, st, 0);
    }
    f32x4 acc[XT][1];
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) acc[xt][0] = zero4();
    float m[1] = {-INFINITY}, lsum[1] = {0.f};
    // The wave's next stage: its K goes out once this one's K has been read, its
    // V once this one's V has, so K and V are in flight together but for the
    // time their tile is read. vmcnt counts in order: NL loads (this stage's V)
    // follow K, NL + 1 (the blocks after next and the next K) follow V.
    for (; st < s_hi; st += NW, ++n) {
        const bool more = st + NW < s_hi, after = st + 2 * NW < s_hi;
        wait_loads<NL>();
        fwd_stage<Pol, 1, true, true, false, true>(
            acc, m, lsum, qf, sk, sv, st * 64, qpos - l16, Nk, g, l16, p.scale_log2,
            [&]() __attribute__((always_inline)) {
                wait_lds();
                if (more) {
                    // the buffer this stage's blocks were in: its V is out already
                    fetch(after ? st + 2 * NW : st, n);
                    load(sk, K, st + NW, n + 1);
                }
            },
            [&]() __attribute__((always_inline)) {
                if (more) {
                    wait_loads<NL + 1>();
                } else {
                    wait_loads<0>();
                }
            });
        wait_lds();
        if (more) load(sv, V, st + NW, n + 1);
    }
    const float lw = xg_sum(lsum[0]);
    float z = 0.f * lw;
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt][0]);
    const bool bad = __builtin_amdgcn_ballot_w64(z != 0.f) != 0;
    __syncthreads();  // every wave is done with the tiles
    if (tid == 0) sm.merge.bad = 0;
    __syncthreads();
    if (bad && lane == 0) sm.merge.bad = 1;
    if (wave < NW) {
#pragma unroll
        for (int i = 0; i < XT; ++i)
            *reinterpret_cast<f32x4 *>(&sm.merge.acc[own][l16][batch_col<Pol>(i, g)]) = batch_quad<Pol>(acc, i, 0);
        if (g == 0) *reinterpret_cast<float2 *>(sm.merge.ml[own][l16]) = make_float2(m[0], lw);
    }
    __syncthreads();
    float *part = nullptr, *ml = nullptr;
    if (slot >= 0) {
        part = batch_part(p.part[0], slot, ROWS, D);
        ml = batch_ml(p.part[0], few_slots(p), slot, ROWS, D);
    }
    if (sm.merge.bad) {
        if (tid < 4 * ROWS) batch_plain<T, D, ROWS>(p, it, 0, s_lo * 64, s_hi * 64, part, ml);
        return;
    }
    for (int i = tid; i < it.s.rows * (D / 4); i += THREADS) {
        const int r = i / (D / 4), c = 4 * (i % (D / 4));
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm.merge.ml[w][r][0]);
        const float mref = M == -INFINITY ? 0.f : M;  // no key of the row here: weight 0
        f32x4 o = zero4();
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float x = fast_exp2(sm.merge.ml[w][r][0] - mref);
            L += x * sm.merge.ml[w][r][1];
            o += *reinterpret_cast<const f32x4 *>(&sm.merge.acc[w][r][c]) * x;
        }
        if (part != nullptr) {
            store4<float>(part + r * D + c, o, 1.0f);
            if (c == 0) *reinterpret_cast<float2 *>(ml + 2 * r) = make_float2(M, L);
        } else {
            batch_store<T>(p, it, r, D, c, o, M, L);
        }
    }
}

// Work-group g of the few-row form: KV head g % Hkv, run g / Hkv of its line. Equal
// runs, one work-group to a CU (its tiles take the LDS): 64 sequences of 2000-16384
// positions, 32/8 heads, d = 128, in 393 us with the join, at the step that brought
// them, 415 with a work-group per share of a sequence, whose count the host can only
// bound: thousands are empty.
template <class Pol, int NW, int THREADS>
__device__ __forceinline__ void batch_few_body(const BatchParams &p, int g, BatchFewSmem<Pol, NW> &sm) {
    const unsigned all = few_line(p), run = few_run(p, all);
    unsigned x = (unsigned)(g / p.Hkv) * run;
    const unsigned x1 = min(x + run, all);
    // what the join of a sequence that the run ends in reads
    auto note = [&](const FewNote &n) __attribute__((always_inline)) {
        if (threadIdx.x == 0 && p.few_groups > 1) reinterpret_cast<FewNote *>(p.notes[0])[g] = n;
    };
    if (x >= x1) return note(FewNote{0, 0, 0, 0});
    BatchItem it;
    it.head = g % p.Hkv;
    it.unit = 0;
    few_walk(p, x, [&](int seq, const BatchSeq &s, unsigned u0, unsigned u1) __attribute__((always_inline)) {
        it.seq = seq;
        it.s = s;
        const FewPiece f = few_piece(x, x1, u0, u1, g);
        if (f.end >= x1) note(FewNote{f.slot == 2 * g + 1 ? few_parts(run, u0, u1) : 0, s.q0, s.rows, s.pos});
        batch_few_piece<Pol, NW, THREADS>(p, it, f.lo, f.hi, f.slot, sm);
        x = f.end;
        if (x < x1) __syncthreads();  // the next piece's tiles are this one's join
        return x >= x1;
    });
}

// ----------------------------------------------------------------- the many rows

template <class Pol>
struct BatchManySmem {
    typename Pol::T k[2][Pol::ROWS * Pol::D], v[2][Pol::ROWS * Pol::D];
    int bad[4];
};

// One unit's share, 16 QT rows per wave: K and V double-buffered in LDS, staged by
// all four waves and read by each. The last 2048 of 32768 tokens, 32/8 heads, d = 128: 960
// us, 1110 TFLOP/s, the matrix units busy in half of the cycles, at 1.9 GHz.
template <class Pol, int QT>
__device__ __forceinline__ void batch_many_body(const BatchParams &p, int block, BatchManySmem<Pol> &sm) {
    using T = typename Pol::T;
    using Stage = BatchStage<Pol, 256>;
    constexpr int D = Pol::D, XT = D / 16, BK = Pol::ROWS, ROWS = 64 * QT;
    constexpr bool kPrio = true;
    auto &sK = sm.k;
    auto &sV = sm.v;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    BatchItem it;
    if (!find_item<ROWS>(p, batch_order(p, block), it)) return;
    const T *K = static_cast<const T *>(p.k) + it.head * D, *V = static_cast<const T *>(p.v) + it.head * D;

    const int r0 = it.unit * ROWS, rw = r0 + wave * 16 * QT;  // the unit's and the wave's first row
    const int last_row = it.s.rows - 1;
    RowPos<QT> qpos;
    typename Pol::Frag qf[QT][Pol::NC];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = min(rw + 16 * qt + l16, last_row);
        qpos.at[qt] = it.s.pos + row / p.group;
        row_frags<Pol>(qf[qt], static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D), g);
    }
    // positions of the unit's first and last row, and of the wave's last
    const int pos_lo = it.s.pos + r0 / p.group;
    const int pos_hi = it.s.pos + min(r0 + ROWS - 1, last_row) / p.group;
    const int pos_w = it.s.pos + min(rw + 16 * QT - 1, last_row) / p.group;
    f32x4 acc[XT][QT];
    float m[QT], lsum[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) acc[xt][qt] = zero4();
        m[qt] = -INFINITY;
        lsum[qt] = 0.f;
    }

    const int Nk = min(it.s.keys, max(pos_hi + 1, 0)), n = (Nk + BK - 1) / BK;
    const BatchRows rows{p.table + (long long)it.seq * p.table_stride, p.bs_shift, Nk, (unsigned)(p.n_blocks - 1)};
    const typename Stage::Stride stride = Stage::stride_bytes(p.kv_rs);
    int s_lo, s_hi;
    share_stages(it, n, s_lo, s_hi);
    // each wave's lanes hold the blocks of the 64 rows of the stage to be staged
    // next, fetched a stage ahead, and pass the cache rows on where a load needs
    // them
    int blk = 0;
    auto fetch = [&](int st) __attribute__((always_inline)) { blk = rows.table[rows.block_at(st * BK + lane)]; };
    auto stage_next = [&](T *sk, T *sv, int st) __attribute__((always_inline)) {
        const unsigned mine = rows.row(blk, st * BK + lane);
        Stage stage;
        stage.rows(tid, stride, [&](int r) __attribute__((always_inline)) { return (unsigned)__shfl((int)mine, r, 64); });
        stage.load(sk, K, wave);
        stage.load(sv, V, wave);
        if (st + 1 < s_hi) fetch(st + 1);
    };
    if (s_lo < s_hi) {
        fetch(s_lo);
        stage_next(sK[0], sV[0], s_lo);
    }
    wait_stage();
    __syncthreads();
    // stages before `whole` hold no key that a row of the unit does not see: in
    // pairs, the LDS buffer a compile-time constant (fwd_entry's reasons)
    const int whole = min(s_hi, min(Nk, pos_lo + 1) / BK);
    const bool some = rw <= last_row;  // the wave has rows
    auto main_stage = [&](auto buf, auto first, int st) __attribute__((always_inline)) {
        constexpr int B = decltype(buf)::value;
        if (st + 1 < s_hi) stage_next(sK[B ^ 1], sV[B ^ 1], st + 1);
        if (some) {
            if constexpr (decltype(first)::value) {
                fwd_stage<Pol, QT, true, false, kPrio>(acc, m, lsum, qf, sK[B], sV[B], st * BK, qpos, Nk, g, l16,
                                                       p.scale_log2);
            } else {
                fwd_stage_lazy<Pol, QT, true, false, kPrio>(acc, m, lsum, qf, sK[B], sV[B], st * BK, qpos, Nk, g, l16,
                                                            p.scale_log2);
            }
        }
        wait_stage();
        __syncthreads();
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    int st = s_lo;
    if (st < whole) main_stage(B0{}, std::true_type{}, st++);
    for (; st + 1 < whole; st += 2) {
        main_stage(B1{}, std::false_type{}, st);
        main_stage(B0{}, std::false_type{}, st + 1);
    }
    if (st < whole) main_stage(B1{}, std::false_type{}, st++);
    for (; st < s_hi; ++st) {
        const int cur = (st - s_lo) & 1;
        if (st + 1 < s_hi) stage_next(sK[cur ^ 1], sV[cur ^ 1], st + 1);
        if (some && st * BK <= pos_w)  // else no row of the wave sees the stage
            fwd_stage<Pol, QT, true, true, kPrio, true>(acc, m, lsum, qf, sK[cur], sV[cur], st * BK, qpos, Nk, g, l16,
                                                        p.scale_log2);
        wait_stage();
        __syncthreads();
    }
    float ltot[QT], z = 0.f;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        ltot[qt] = xg_sum(lsum[qt]);
        z += 0.f * ltot[qt];
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt][qt]);
    }
    float *part = nullptr, *ml = nullptr;
    if (it.shares > 1) {
        part = batch_part(p.part[1], it.slot, ROWS, D);
        ml = batch_ml(p.part[1], p.slots, it.slot, ROWS, D);
    }
    const bool bad = __builtin_amdgcn_ballot_w64(z != 0.f) != 0;
    if (lane == 0) sm.bad[wave] = bad;
    __syncthreads();
    if (sm.bad[0] | sm.bad[1] | sm.bad[2] | sm.bad[3]) {
        for (int i = 0; i < QT; ++i) batch_plain<T, D, ROWS>(p, it, 64 * i, s_lo * BK, s_hi * BK, part, ml);
        return;
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = rw + 16 * qt + l16, rl = r - r0;
        const bool have = r < it.s.rows;
        if (it.shares > 1) {
            if (have) {
#pragma unroll
                for (int i = 0; i < XT; ++i)
                    store4<float>(part + rl * D + batch_col<Pol>(i, g), batch_quad<Pol>(acc, i, qt), 1.0f);
                if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * rl) = make_float2(m[qt], ltot[qt]);
            }
            continue;
        }
        const float inv = batch_inverse(ltot[qt], qpos.at[qt]);
        T *O = static_cast<T *>(p.o) + batch_elem(p, it, min(r, last_row), p.o_rs, D);
#pragma unroll
        for (int xt = 0; xt < XT; xt += 2)
            store8_pair_bf16(O, 16 * xt, g, acc[xt][qt], acc[xt + 1][qt], inv, have);
        if (p.lse != nullptr && have && g == 0)
            p.lse[batch_lse(p, it, r)] = ltot[qt] > 0.f ? (m[qt] + fast_log2(ltot[qt])) * kLn2 : -INFINITY;
    }
}

// The same for fp32 (d = 64), 16 rows per wave of 8, with its products in bf16 parts
// (Split3): K and V pass through registers, loaded one stage ahead, and are
// split once per work-group into one LDS buffer; two work-groups per CU. Operands
// that the parts cannot hold (kPartMin, infinities) flag the unit, whose rows
// are then run in plain arithmetic. Bound by the splitting beside the products. us,
// 2000 tokens of 14/2 heads after 2096: 177 (matrix units busy 33%); at the step that
// brought it 176, 203 with 4 waves and 64 rows, 235 on v_mfma_f32_16x16x4_f32.
__device__ __forceinline__ void batch_many_parts(const BatchParams &p, int block, FwdSplitSmem &sm) {
    constexpr int D = 64, XT = 4, BK = 64, NW = kBatchF32Waves, NT = 64 * NW, ROWS = 16 * NW;
    using PL = PolBF16<64>;  // the parts' layout
    using Stage = SplitStage<NT>;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    BatchItem it;
    if (!find_item<ROWS>(p, batch_order(p, block), it)) return;
    const float *K = static_cast<const float *>(p.k) + it.head * D, *V = static_cast<const float *>(p.v) + it.head * D;

    const int r0 = it.unit * ROWS, rw = r0 + wave * 16, r = rw + l16;
    const int last_row = it.s.rows - 1, row = min(r, last_row);
    const int qpos = it.s.pos + row / p.group;
    const int pos_lo = it.s.pos + r0 / p.group;
    const int pos_hi = it.s.pos + min(r0 + ROWS - 1, last_row) / p.group;
    const int pos_w = it.s.pos + min(rw + 15, last_row) / p.group;
    const int Nk = min(it.s.keys, max(pos_hi + 1, 0)), n = (Nk + BK - 1) / BK;
    const BatchRows rows{p.table + (long long)it.seq * p.table_stride, p.bs_shift, Nk, (unsigned)(p.n_blocks - 1)};
    int s_lo, s_hi;
    share_stages(it, n, s_lo, s_hi);

    // this thread's chunks of a tile: row and first column
    int srow[Stage::NK], scol[Stage::NK];
#pragma unroll
    for (int k = 0; k < Stage::NK; ++k) {
        PL::chunk_at(k * NT + tid, srow[k], scol[k]);
        scol[k] *= 8;
    }
    int blk = 0;  // of the lane's row of the stage to be loaded next
    auto fetch = [&](int st) __attribute__((always_inline)) { blk = rows.table[rows.block_at(st * BK + lane)]; };
    Stage xk, xv;
    auto load = [&](int st) __attribute__((always_inline)) {
        const unsigned mine = rows.row(blk, st * BK + lane);
#pragma unroll
        for (int k = 0; k < Stage::NK; ++k) {
            const unsigned at = (unsigned)__shfl((int)mine, srow[k], 64);
            const size_t off = (size_t)at * (size_t)p.kv_rs + scol[k];
            xk.load(k, K + off);
            xv.load(k, V + off);
        }
        if (st + 1 < s_hi) fetch(st + 1);
    };
    if (s_lo < s_hi) {
        fetch(s_lo);
        load(s_lo);
    }
    Split3 qf[1][2];
    const bool low = split_row(qf[0], static_cast<const float *>(p.q) + batch_elem(p, it, row, p.q_rs, D), g,
                               p.scale_log2 * kPartDown, r <= last_row);
    f32x4 acc[XT][1];
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) acc[xt][0] = zero4();
    float m = -INFINITY, lsum = 0.f;

    // One stage: the share's first, or m raised only where a lane's sum of p
    // passes kLazySum. A row that sees no key of the first stage keeps m = -inf,
    // and sees none of the later ones.
    auto compute = [&](auto first, bool edge, int k0) __attribute__((always_inline)) {
        constexpr bool FIRST = decltype(first)::value;
        f32x4 s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Split3 a[1][2];
                f32x4 c[1][1] = {{zero4()}};
                sm.k.row_frags(a[0], 32 * u + PL::arow(t, l16), g);
                mma_split_tiles<2, 1, 1>(c, a, qf);
                s[u][t] = c[0][0];
            }
        }
        if (edge) {
            const int lim = min(qpos, Nk - 1) - k0 - PL::bidx(0, g, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (32 * u + PL::bidx(t, 0, e) > lim) s[u][t][e] = -INFINITY;
                    }
                }
            }
        }
        const float base = m == -INFINITY ? 0.f : m;  // what p is relative to
        f32x4 pv[2][2];
        auto exps = [&](float sub) __attribute__((always_inline)) {
            float ls = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = fast_exp2(s[u][t][e] - sub);
                        pv[u][t][e] = x;
                        ls += x;
                    }
                }
            }
            return ls;
        };
        auto raise = [&]() __attribute__((always_inline)) {
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[u][t][e]);
                }
            }
            mx = fmaxf(xg_max(mx), m);
            const float to = mx == -INFINITY ? 0.f : mx;
            if constexpr (!FIRST) {
                const float corr = fast_exp2(base - to);
                lsum *= corr;
#pragma unroll
                for (int xt = 0; xt < XT; ++xt) acc[xt][0] *= corr;
            }
            m = mx;
            lsum += exps(to);
        };
        if constexpr (FIRST) {
            raise();
        } else {
            const float ls = exps(base);
            if (__builtin_amdgcn_ballot_w64(ls > kLazySum) != 0) {
                raise();
            } else {
                lsum += ls;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const Split3 pf[1] = {split3(pv[u][0], pv[u][1])};
#pragma unroll
            for (int xt = 0; xt < XT; ++xt) {
                const Split3 a[1] = {sm.v.chain_a(16 * xt, 32 * u, g, l16)};
                acc[xt][0] = mma_split<1>(a, pf, acc[xt][0]);
            }
        }
    };
    // stages before `whole` hold no key that a row of the unit does not see
    const int whole = min(s_hi, min(Nk, pos_lo + 1) / BK);
    auto stage = [&](auto first, int st) __attribute__((always_inline)) {
        if (st > s_lo) barrier_lds();  // every wave is done with the stage before
        xk.write(sm.k, tid);
        xv.write(sm.v, tid);
        if (st + 1 < s_hi) load(st + 1);
        barrier_lds();
        if (rw <= last_row && st * BK <= pos_w) compute(first, st >= whole, st * BK);
    };
    if (s_lo < s_hi) stage(std::true_type{}, s_lo);
    for (int st = s_lo + 1; st < s_hi; ++st) stage(std::false_type{}, st);
    const float ltot = xg_sum(lsum);
    float z = 0.f * ltot;
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt][0]);
    // a row that sees keys of the share, all of whose scores overflowed to -inf
    if (rw <= last_row && m == -INFINITY && s_lo < s_hi && s_lo * BK <= qpos) z = NAN;
    if (low) z = NAN;
    float *part = nullptr, *ml = nullptr;
    if (it.shares > 1) {
        part = batch_part(p.part[1], it.slot, ROWS, D);
        ml = batch_ml(p.part[1], p.slots, it.slot, ROWS, D);
    }
    if (any_nonfinite<NW>(z, sm.flags, wave, lane)) {
        batch_plain<float, D, ROWS>(p, it, 0, s_lo * BK, s_hi * BK, part, ml);
        return;
    }
    if (r > last_row) return;
    if (part != nullptr) {
        const int rl = r - r0;
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) store4<float>(part + rl * D + 16 * xt + 4 * g, acc[xt][0], kPartDown);
        if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * rl) = make_float2(m, ltot);
        return;
    }
    const float inv = ltot > 0.f ? kPartDown / ltot : 0.f;
    float *O = static_cast<float *>(p.o) + batch_elem(p, it, r, p.o_rs, D);
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) store4<float>(O + 16 * xt + 4 * g, acc[xt][0], inv);
    if (p.lse != nullptr && g == 0)
        p.lse[batch_lse(p, it, r)] = ltot > 0.f ? (m + fast_log2(ltot)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------------- the join

// The parts of a unit's rows [first, end): o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s
// - M) l_s, part s being slot at(s) of the workspace, 128 parts at a time. A
// group of D / 4 threads, four elements each, has a row; where there are few
// rows several groups take turns over its parts and meet in LDS. Bound by
// latency: the (max, sum) pairs of all parts are one round of loads, and eight
// parts of a thread's turn another. us, one token after 65535, 14/2 heads (128 parts
// of 7 rows): 6.6; 7.4 when it came, and 11.2 with one group to a row; 28 tokens and 4 chunks: 7.2
// with the notes, 12.8 where each work-group found its unit in the lengths.
template <class T, int D, class At>
__device__ __forceinline__ void batch_join_rows(const BatchParams &p, const BatchItem &it, int rows, int first, int end,
                                                int S, float *parts, int slots, At at) {
    constexpr int C = D / 4, NG = 256 / C, PARTS = 128, EACH = PARTS / C;
    __shared__ __attribute__((aligned(16))) f32x4 so[NG][C];
    __shared__ float weights[NG][PARTS];
    const int tid = threadIdx.x, c = tid % C, grp = tid / C, nrows = end - first;
    int together = 1;  // groups to a row
    while (together * 2 * nrows <= NG) together *= 2;
    const int turn = grp % together;
    for (int r0 = 0; r0 < nrows; r0 += NG / together) {
        const bool have = r0 + grp / together < nrows;
        const int r = have ? first + r0 + grp / together : first;  // (others repeat a row and store nothing)
        float M = -INFINITY, L = 0.f;
        f32x4 o = zero4();
        for (int s0 = 0; s0 < S; s0 += PARTS) {
            const int n = min(PARTS, S - s0);
            float2 v[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                v[i] = make_float2(-INFINITY, 0.f);
                if (i * C + c < n)
                    v[i] = *reinterpret_cast<const float2 *>(batch_ml(parts, slots, at(s0 + i * C + c), rows, D) + 2 * r);
            }
            float mx = M;
#pragma unroll
            for (int i = 0; i < EACH; ++i) mx = fmaxf(mx, v[i].x);
#pragma unroll
            for (int k = C / 2; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
            const float mref = mx == -INFINITY ? 0.f : mx, corr = fast_exp2(M - mref);
            M = mx;
            L *= corr;
            o *= corr;
            float l = 0.f;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const float w = fast_exp2(v[i].x - mref);
                l += w * v[i].y;
                weights[grp][i * C + c] = w;  // read by the group's own lanes of the wave
            }
#pragma unroll
            for (int k = C / 2; k > 0; k >>= 1) l += __shfl_xor(l, k, 64);
            L += l;
            wait_lds();
            for (int s = turn; s < n; s += 8 * together) {
                f32x4 x[8];
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int j = min(s + i * together, n - 1);
                    w[i] = s + i * together < n ? weights[grp][j] : 0.f;
                    x[i] = *reinterpret_cast<const f32x4 *>(batch_part(parts, at(s0 + j), rows, D) + r * D + 4 * c);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // (past the last part: its load again, which adds nothing, also where it is infinite)
                    o += (s + i * together < n ? x[i] : zero4()) * w[i];
                }
            }
            wait_lds();
        }
        if (together > 1) {
            __syncthreads();
            so[grp][c] = o;
            __syncthreads();
            if (turn == 0) {
                for (int k = 1; k < together; ++k) o += so[grp + k][c];
            }
        }
        if (have && turn == 0) batch_store<T>(p, it, it.unit * rows + r, D, 4 * c, o, M, L);
    }
}

// Grid: the cuts of the few-row form's lines (the work-groups but the last run's),
// then the pieces of the split units that the many-row form may have.
template <class T, int D>
__device__ __forceinline__ void batch_join(const BatchParams &p, int few_cuts) {
    constexpr int JOIN = join_rows(D);
    const int rows = p.many_rows, pieces = rows / JOIN;
    BatchItem it;
    if ((int)blockIdx.x < few_cuts) {
        // the cut at the end of work-group g's run
        const int heads = p.Hkv, g = (int)blockIdx.x / kFewJoins, first = (int)blockIdx.x % kFewJoins * (kBatchFew / kFewJoins);
        const FewNote n = reinterpret_cast<const FewNote *>(p.notes[0])[g];
        const int end = min(first + kBatchFew / kFewJoins, n.rows);
        if (n.parts < 2 || first >= end) return;
        const int run = g / heads, head = g - run * heads;
        it.head = head;
        it.unit = 0;
        it.s.q0 = n.q0;
        it.s.pos = n.pos;
        batch_join_rows<T, D>(p, it, kBatchFew, first, end, n.parts, p.part[0], few_slots(p), [&](int i) __attribute__((always_inline)) {
            return i == 0 ? few_first_slot(run, heads, head) : few_next_slot(run, heads, head) + 2 * heads * (i - 1);
        });
        return;
    }
    const int w = (int)blockIdx.x - few_cuts, unit = w / pieces;
    const int count = p.notes[1][0];
    const ManyNote n = reinterpret_cast<const ManyNote *>(p.notes[1])[1 + unit];
    if (unit >= count || !note_holds(p, n)) return;
    const int first = w % pieces * JOIN, end = min(first + JOIN, n.rows - n.unit * rows);
    if (first >= end) return;
    it.head = n.head;
    it.unit = n.unit;
    it.s.q0 = n.q0;
    it.s.pos = n.pos[0];
    batch_join_rows<T, D>(p, it, rows, first, end, n.shares, p.part[1], p.slots,
                                [&](int i) __attribute__((always_inline)) { return n.slot + i * p.Hkv; });
}

// Both forms in one launch: the few-row form's work-groups first, each wave's
// tiles a quarter of its work-group's (bf16, d = 64) or half of it, so that LDS
// holds as many of them as of the many-row form's: their reads and its matrix
// products then share the CUs (us, 28 tokens and 4 chunks: 48.6; 41 + 17 in two
// launches). In fp32 the few-row form has to spill 96 at the other's 128 registers;
// two launches took the same (6 tokens and 2 chunks: 13 + 55 and 55).
template <int QT, class Pol>
__device__ __forceinline__ void batch_many(const BatchParams &p, int block, BatchManySmem<Pol> &sm) {
    batch_many_body<Pol, QT>(p, block, sm);
}
template <int QT>
__device__ __forceinline__ void batch_many(const BatchParams &p, int block, FwdSplitSmem &sm) {
    batch_many_parts(p, block, sm);
}
template <class Pol, class Many, int QT, int NW, int THREADS>
__device__ __forceinline__ void batch_both_body(const BatchParams &p, int few_groups) {
    __shared__ __attribute__((aligned(16))) union {
        BatchFewSmem<Pol, NW> few;
        Many many;
    } sm;
    if ((int)blockIdx.x < few_groups) {
        batch_few_body<Pol, NW, THREADS>(p, blockIdx.x, sm.few);
    } else {
        batch_many<QT>(p, (int)blockIdx.x - few_groups, sm.many);
    }
}

// (MANY: of units of 64 QT rows, WPS waves per SIMD)
#define MXFA_BATCH_MANY(NAME, BOTH, POL, MANY, QT, THREADS, WPS, BOTH_NW, BOTH_WPS)                          \
    extern "C" __global__ __launch_bounds__(THREADS, WPS) void mxfa_batch_##NAME(BatchParams p) {            \
        __shared__ __attribute__((aligned(16))) MANY sm;                                                     \
        batch_many<QT>(p, blockIdx.x, sm);                                                                   \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(THREADS, BOTH_WPS) void mxfa_batch_##BOTH(BatchParams p, int few_groups) { \
        batch_both_body<POL, MANY, QT, BOTH_NW, THREADS>(p, few_groups);                                     \
    }
#define MXFA_BATCH(SUFFIX, POL, NW)                                                                          \
    extern "C" __global__ __launch_bounds__(64 * NW) void mxfa_batch_##SUFFIX##_few(BatchParams p) {         \
        __shared__ __attribute__((aligned(16))) BatchFewSmem<POL, NW> sm;                                    \
        batch_few_body<POL, NW, 64 * NW>(p, blockIdx.x, sm);                                                 \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(256) void mxfa_batch_##SUFFIX##_join(BatchParams p, int few_groups) { \
        batch_join<POL::T, POL::D>(p, few_groups);                                                           \
    }
MXFA_BATCH(b64, PolRows<64>, 8)
MXFA_BATCH_MANY(b64_many, b64_both, PolRows<64>, BatchManySmem<PolRows<64>>, 2, 256, 3, 3, 3)
MXFA_BATCH_MANY(b64_many64, b64_both64, PolRows<64>, BatchManySmem<PolRows<64>>, 1, 256, 4, 3, 3)
MXFA_BATCH(b128, PolRows<128>, 4)
MXFA_BATCH_MANY(b128_many, b128_both, PolRows<128>, BatchManySmem<PolRows<128>>, 2, 256, 2, 2, 2)
MXFA_BATCH_MANY(b128_many64, b128_both64, PolRows<128>, BatchManySmem<PolRows<128>>, 1, 256, 2, 2, 2)
MXFA_BATCH(f64, PolF32, 4)
MXFA_BATCH_MANY(f64_many, f64_both, PolF32, FwdSplitSmem, 2, 64 * kBatchF32Waves, 4, 2, 4)
#undef MXFA_BATCH_MANY
#undef MXFA_BATCH
#endif

// The forms of a call; groups = 0: not launched.
static void batch_forms(BatchParams *p, int dtype_bf16, BatchForm (&f)[2]) {
    batch_plan(p, dtype_bf16);
    f[0] = f[1] = BatchForm{0, 0, 0, 0, 0};
    if (p->few_rows > 0) f[0] = batch_few_form(p);
    if (batch_may_be_many(*p)) f[1] = batch_many_form(p, dtype_bf16);
}

size_t batch_workspace_bytes(const BatchParams &q, int dtype_bf16) {
    BatchParams p = q;
    BatchForm f[2];
    batch_forms(&p, dtype_bf16, f);
    size_t n = 0;
    for (const BatchForm &x : f) n += batch_slot_floats(x.slots, x.rows, p.d) + (size_t)x.notes;
    return std::max<size_t>(n * sizeof(float), 16);
}

long long batch_groups(const BatchParams &q, int dtype_bf16) {
    BatchParams p = q;
    batch_plan(&p, dtype_bf16);
    return std::max(batch_few_form(&p).groups, batch_many_form(&p, dtype_bf16).groups);
}

hipError_t launch_batch(BatchParams p, int dtype_bf16, void *workspace, hipStream_t stream) {
    static constexpr KernelId ids[3][6] = {
        {k_mxfa_batch_b64_few, k_mxfa_batch_b64_join, k_mxfa_batch_b64_many, k_mxfa_batch_b64_both,
         k_mxfa_batch_b64_many64, k_mxfa_batch_b64_both64},
        {k_mxfa_batch_b128_few, k_mxfa_batch_b128_join, k_mxfa_batch_b128_many, k_mxfa_batch_b128_both,
         k_mxfa_batch_b128_many64, k_mxfa_batch_b128_both64},
        {k_mxfa_batch_f64_few, k_mxfa_batch_f64_join, k_mxfa_batch_f64_many, k_mxfa_batch_f64_both}};
    const KernelId *id = ids[!dtype_bf16 ? 2 : p.d == 128 ? 1 : 0];
    BatchForm f[2];
    batch_forms(&p, dtype_bf16, f);
    const KernelId *many = id + (p.many_rows == 64 ? 4 : 2);
    float *next = static_cast<float *>(workspace);
    for (int i = 0; i < 2; ++i) {  // (notes of 16 and 32 bytes, slots of a multiple of that)
        p.part[i] = next;
        next += batch_slot_floats(f[i].slots, f[i].rows, p.d);
        p.notes[i] = reinterpret_cast<int *>(next);
        next += f[i].notes;
    }
    const int threads = dtype_bf16 ? 256 : 64 * kBatchF32Waves;
    hipError_t e;
    int few_groups = (int)f[0].groups;
    void *args[] = {&p, &few_groups};
    if (f[1].groups == 0) {
        e = launch_kernel(id[0], dim3(few_groups), dim3(dtype_bf16 && p.d == 64 ? 512 : 256), args, stream);
    } else if (few_groups == 0) {
        e = launch_kernel(many[0], dim3((unsigned)f[1].groups), dim3(threads), args, stream);
    } else {
        e = launch_kernel(many[1], dim3((unsigned)(few_groups + f[1].groups)), dim3(threads), args, stream);
    }
    int cuts = (int)f[0].joins * kFewJoins;
    const unsigned joins = (unsigned)(cuts + f[1].joins * (f[1].rows / join_rows(p.d)));
    if (e != hipSuccess || joins == 0) return e;
    void *jargs[] = {&p, &cuts};
    return launch_kernel(id[1], dim3(joins), dim3(256), jargs, stream);
}

}  // namespace mxfa
