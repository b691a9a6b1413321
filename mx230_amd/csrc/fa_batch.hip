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
// group. Two forms take them in units of rows:
//   * few (at most 16 rows): every wave holds the same rows and takes 64-key
//     stages of its own; bound by the reads of K and V;
//   * many: 64 rows, 16 per wave, the waves sharing each stage; bound by the
//     matrix products.
// The host knows neither lengths nor units: a work-group finds its item (a
// unit's share of its keys) from cu_q and lens itself (find_item). A unit is
// split over its keys where the whole work, spread over the target count of
// items, gives each less than the unit has; its shares' unnormalised outputs
// are then joined by a second launch, in a fixed order.
#include <algorithm>
#include <climits>

#include "fa_cache.h"
#include "fa_device.h"
#include "fa_launch.h"

namespace mxfa {

constexpr int kBatchFew = 16, kBatchMany = 64;  // rows of a unit
// the fewest stages of a share, per form: shorter ones cost more in the join
// than they save
constexpr int kFewLeast = 4, kManyLeast = 4;

template <bool FEW>
constexpr int batch_rows() {
    return FEW ? kBatchFew : kBatchMany;
}
template <bool FEW>
constexpr int batch_least() {
    return FEW ? kFewLeast : kManyLeast;
}
// Slots of the workspace: the shares of split units. A unit of n stages is
// split where n > quota, into ceil(n / quota) < 2 n / quota shares, and quota
// >= all stages / target, so there are at most 2 target of them.
__host__ __device__ constexpr long long batch_slots(int target) { return 2LL * target; }
__host__ __device__ constexpr size_t batch_part_floats(int target, int rows, int d) {
    return (size_t)batch_slots(target) * rows * (d + 2);
}

// ------------------------------------------------- fp32 on its own instructions

// fp32 inputs (d = 64) on v_mfma_f32_16x16x4_f32, in the policy form of
// fwd_stage. LDS rows of 256 bytes hold their 16-byte chunk c at c ^ (row & 15),
// so the 16 rows of a score operand and the 16 chunks of a V row both cover
// all banks. Score k-steps: MFMA (c, e) takes element 16c + 4g + e of lane
// group g. In the chained product a lane reads 4 columns of a V row at once, so
// tile xt's row 4g + r of O^T is column 4 (4g + r) + xt.
struct PolF32 {
    static constexpr int D = 64;
    using T = float;
    using Frag = f32x4;
    static constexpr int EPC = 4, NC = 4, ROWS = 64;
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

// A row's elements that a lane holds as operand B of the scores.
template <class Pol>
__device__ __forceinline__ void row_frags(typename Pol::Frag (&f)[Pol::NC], const typename Pol::T *row, int g) {
    constexpr int S = sizeof(typename Pol::T) == 2 ? 8 : 4;
#pragma unroll
    for (int c = 0; c < Pol::NC; ++c) f[c] = *reinterpret_cast<const typename Pol::Frag *>(row + 4 * S * c + S * g);
}

// ------------------------------------------------------------- staging of pages

// A sequence's stages of keys into LDS, NT threads to a tile; keys past the
// last count as the last, and blocks outside the pool as the nearest in it, so
// no read leaves the caches.
template <class Pol, int NT>
struct BatchStage {
    RowPlan<Pol, NT> plan;
    PagedRows<Pol, NT> rows;
    static constexpr int LOADS = RowPlan<Pol, NT>::NK;
    __device__ explicit BatchStage(int tid) : plan(tid) {}
    __device__ __forceinline__ void fetch(const int *table, int shift, unsigned last_block, int k0, int Nk) {
        rows.fetch(table, shift, k0, Nk, plan);
#pragma unroll
        for (int r = 0; r < PagedRows<Pol, NT>::NR; ++r) rows.blk[r] = (int)min((unsigned)rows.blk[r], last_block);
    }
    __device__ __forceinline__ void load(typename Pol::T *tile, const typename Pol::T *X, int k0, int Nk, int shift,
                                         int wave, int stride) const {
        rows.stage_one(tile, X, k0, Nk, shift, plan, wave, stride);
    }
};
// fp32: a load of NT threads covers NT / 16 whole rows. Each wave's lanes hold
// the blocks of the stage's 64 rows, passed on where a load needs them.
template <int NT>
struct BatchStage<PolF32, NT> {
    static constexpr int LOADS = 64 * 16 / NT;
    int tid, blk;
    __device__ explicit BatchStage(int t) : tid(t), blk(0) {}
    __device__ __forceinline__ void fetch(const int *table, int shift, unsigned last_block, int k0, int Nk) {
        blk = (int)min((unsigned)table[min(k0 + (tid & 63), Nk - 1) >> shift], last_block);
    }
    __device__ __forceinline__ void load(float *tile, const float *X, int k0, int Nk, int shift, int wave,
                                         int stride) const {
        const uint32_t base = lds_addr(tile) + wave * 64 * 16;
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            const int row = (k * NT + tid) >> 4, c = (tid & 15) ^ (row & 15);
            const int b = __shfl(blk, row, 64), t = min(k0 + row, Nk - 1);
            const size_t at = (((size_t)b << shift) + (size_t)(t & ((1 << shift) - 1))) * (size_t)stride;
            lds_dma16(base + k * NT * 16, X + at + 4 * c);
        }
    }
};

// -------------------------------------------------------------------- the items

// What a sequence brings to a form.
struct BatchSeq {
    int q0;      // its first row of q
    int pos;     // position of that row's token
    int rows;    // new tokens x query heads per KV head (0: none for this form)
    int keys;    // positions that its last token sees
    int units, stages;
};

template <bool FEW>
__device__ __forceinline__ BatchSeq batch_seq(const BatchParams &p, int s) {
    BatchSeq b{0, 0, 0, 0, 0, 0};
    if (s >= p.n_seq) return b;
    const int c0 = p.cu_q[s], c1 = p.cu_q[s + 1], len = p.lens[s];
    b.q0 = min(max(c0, 0), p.n_tok);
    const int count = min(min(c1, p.n_tok) - b.q0, p.max_q);
    // positions stay within int with a stage to spare, whatever the arrays hold
    const long long cap = min((long long)p.max_blocks << p.bs_shift, (long long)INT_MAX - 256);
    const long long pos = (long long)len - ((long long)c1 - b.q0);
    b.pos = (int)min(max(pos, -(1LL << 30)), cap);
    const long long rows = (long long)max(count, 0) * p.group;
    const bool mine = FEW ? rows <= p.few_rows : rows > p.few_rows;
    b.rows = mine ? (int)rows : 0;
    b.keys = (int)min(min((long long)b.pos + max(count, 0), (long long)len), cap);
    b.keys = max(b.keys, 0);
    b.units = (b.rows + batch_rows<FEW>() - 1) / batch_rows<FEW>();
    b.stages = (b.keys + 63) / 64;
    return b;
}

__device__ __forceinline__ long long wave_sum(long long x) {
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) x += __shfl_xor(x, k, 64);
    return x;
}
__device__ __forceinline__ int wave_prefix(int x, int lane) {  // inclusive
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int o = __shfl_up(x, k, 64);
        if (lane >= k) x += o;
    }
    return x;
}

struct BatchItem {
    BatchSeq s;
    int seq, head, unit, share, shares;
    int slot;  // of share 0 (the join) or of this share, where shares > 1
};

// Item `w` of a form (JOIN: split unit `w`), found by every wave for itself: a
// lane per sequence, twice over them where there are more than 64. False past
// the last one. Items of a sequence: units (the last, heaviest one first) x
// shares x KV heads, so that neighbouring work-groups, which the dispatcher
// spreads over the XCDs, have the heads and an XCD's share of them the same
// head's keys.
template <bool FEW, bool JOIN>
__device__ __forceinline__ bool find_item(const BatchParams &p, int w, BatchItem &it) {
    const int lane = threadIdx.x & 63;
    BatchSeq b = batch_seq<FEW>(p, lane);
    long long all = (long long)b.units * max(b.stages, 1);
    for (int s0 = 64; s0 < p.n_seq; s0 += 64) {
        const BatchSeq c = batch_seq<FEW>(p, s0 + lane);
        all += (long long)c.units * max(c.stages, 1);
    }
    all = wave_sum(all) * p.Hkv;
    const int target = p.target[FEW ? 0 : 1];
    const long long quota = max((all + target - 1) / target, (long long)batch_least<FEW>());
    int before = 0, slots = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        if (s0 > 0) b = batch_seq<FEW>(p, s0 + lane);
        const int shares = (long long)b.stages > quota ? (int)((b.stages + quota - 1) / quota) : 1;
        const int per = JOIN ? (shares > 1 ? b.units * p.Hkv : 0) : b.units * p.Hkv * shares;
        const int mine = shares > 1 ? b.units * p.Hkv * shares : 0;
        const int upto = wave_prefix(per, lane), slots_upto = wave_prefix(mine, lane);
        const unsigned long long at = __builtin_amdgcn_ballot_w64(before + upto > w);
        if (at != 0) {
            const int l = __builtin_ctzll(at);
            it.seq = s0 + l;
            it.s.q0 = __builtin_amdgcn_readlane(b.q0, l);
            it.s.pos = __builtin_amdgcn_readlane(b.pos, l);
            it.s.rows = __builtin_amdgcn_readlane(b.rows, l);
            it.s.keys = __builtin_amdgcn_readlane(b.keys, l);
            it.s.units = __builtin_amdgcn_readlane(b.units, l);
            it.s.stages = __builtin_amdgcn_readlane(b.stages, l);
            it.shares = __builtin_amdgcn_readlane(shares, l);
            int i = w - before - __builtin_amdgcn_readlane(upto - per, l);
            it.slot = slots + __builtin_amdgcn_readlane(slots_upto - mine, l);
            if (JOIN) {
                it.slot += i / p.Hkv * it.shares * p.Hkv + i % p.Hkv;  // the unit's shares are Hkv apart
                it.share = 0;
            } else {
                it.slot += i;
            }
            it.head = i % p.Hkv;
            i /= p.Hkv;
            if (!JOIN) {
                it.share = i % it.shares;
                i /= it.shares;
            }
            it.unit = it.s.units - 1 - i;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slots_upto, 63);
    }
    return false;
}

// Row r of a unit's sequence: its elements in q or o, and its index in lse.
__device__ __forceinline__ size_t batch_elem(const BatchParams &p, const BatchItem &it, int r, int stride, int d) {
    return (size_t)(it.s.q0 + r / p.group) * (size_t)stride + (size_t)(it.head * p.group + r % p.group) * d;
}
__device__ __forceinline__ size_t batch_lse(const BatchParams &p, const BatchItem &it, int r) {
    return (size_t)(it.s.q0 + r / p.group) * p.Hq + it.head * p.group + r % p.group;
}

// Four elements of a finished row, and its lse by the row's first thread.
template <class T>
__device__ __forceinline__ void batch_store(const BatchParams &p, const BatchItem &it, int r, int d, int c, f32x4 o,
                                            float m, float l) {
    T *O = static_cast<T *>(p.o) + batch_elem(p, it, r, p.o_rs, d) + c;
    store4<T>(O, o, l > 0.f || l != l ? 1.0f / l : 0.f);  // a row that sees no key is zeros
    if (p.lse != nullptr && c == 0) p.lse[batch_lse(p, it, r)] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

// The columns a lane holds of its row: 4 of them from batch_col(i, g), i < XT.
template <class Pol>
__device__ __forceinline__ int batch_col(int i, int g) {
    return sizeof(typename Pol::T) == 2 ? 16 * i + 4 * g : 16 * g + 4 * i;
}
template <class Pol, int XT>
__device__ __forceinline__ f32x4 batch_quad(const f32x4 (&acc)[XT][1], int i) {
    if constexpr (sizeof(typename Pol::T) == 2) {
        return acc[i][0];
    } else {
        return f32x4{acc[0][0][i], acc[1][0][i], acc[2][0][i], acc[3][0][i]};
    }
}

// A unit's share in plain fp32 arithmetic, keys a row does not see left out
// altogether: taken where a value was not finite, since in the matrix products
// an infinity or NaN in the V of a key that a row does not see reaches it as 0
// x inf. 4 threads per row. o: a row's running (max, sum) and output go where
// the form's would: to the workspace slot, or finished.
template <class T, int D, int ROWS>
__device__ __forceinline__ void batch_plain(const BatchParams &p, const BatchItem &it, int key0, int key1, float *part,
                                            float *ml) {
    constexpr int E = D / 4;
    const int tid = threadIdx.x;
    if (tid >= 4 * ROWS) return;
    const int r = it.unit * ROWS + (tid >> 2), c = E * (tid & 3);
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
        if (it.shares > 1) {
            store4<float>(part + (size_t)(tid >> 2) * D + c + e, o, 1.0f);
        } else {
            batch_store<T>(p, it, r, D, c + e, o, m, l);
        }
    }
    if (it.shares > 1 && c == 0) *reinterpret_cast<float2 *>(ml + 2 * (tid >> 2)) = make_float2(m, l);
}

// The workspace of an item's share: ROWS rows of D floats, and their (max, sum).
template <bool FEW>
__device__ __forceinline__ float *batch_part(const BatchParams &p, int slot, int d) {
    return p.part[FEW ? 0 : 1] + (size_t)slot * batch_rows<FEW>() * d;
}
template <bool FEW>
__device__ __forceinline__ float *batch_ml(const BatchParams &p, int slot, int d) {
    return p.part[FEW ? 0 : 1] + (size_t)batch_slots(p.target[FEW ? 0 : 1]) * batch_rows<FEW>() * d +
           (size_t)slot * batch_rows<FEW>() * 2;
}

// ------------------------------------------------------------------ the few rows

template <class Pol, int NW>
union BatchFewSmem {
    struct {
        typename Pol::T k[NW][Pol::ROWS * Pol::D], v[NW][Pol::ROWS * Pol::D];
    } t;
    struct {
        float acc[NW][kBatchFew][Pol::D + 4];
        float ml[NW][kBatchFew][2];
        int bad;
    } merge;
};

// Each of the NW waves takes every NW-th stage of the share, staged into its
// own tiles with no barrier; the waves' maxima, sums and O meet in LDS.
template <class Pol, int NW>
__device__ __forceinline__ void batch_few_body(const BatchParams &p) {
    using T = typename Pol::T;
    constexpr int D = Pol::D, XT = D / 16;
    __shared__ __attribute__((aligned(16))) BatchFewSmem<Pol, NW> sm;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    BatchItem it;
    if (!find_item<true, false>(p, blockIdx.x, it)) return;
    const T *K = static_cast<const T *>(p.k) + it.head * D, *V = static_cast<const T *>(p.v) + it.head * D;
    const int *table = p.table + (long long)it.seq * p.table_stride;
    const unsigned last_block = p.n_blocks - 1;
    T *sk = sm.t.k[wave], *sv = sm.t.v[wave];
    const int Nk = it.s.keys, n = it.s.stages;
    const int s_lo = (int)((long long)it.share * n / it.shares), s_hi = (int)((long long)(it.share + 1) * n / it.shares);

    BatchStage<Pol, 64> stage(lane);
    constexpr int NL = BatchStage<Pol, 64>::LOADS;
    int st = s_lo + wave;
    if (st < s_hi) {
        stage.fetch(table, p.bs_shift, last_block, st * 64, Nk);
        stage.load(sk, K, st * 64, Nk, p.bs_shift, 0, p.kv_rs);
        stage.load(sv, V, st * 64, Nk, p.bs_shift, 0, p.kv_rs);
    }
    const int row = min(l16, it.s.rows - 1);
    const int qpos = it.s.pos + row / p.group;
    typename Pol::Frag qf[1][Pol::NC];
    row_frags<Pol>(qf[0], static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D), g);
    f32x4 acc[XT][1];
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) acc[xt][0] = zero4();
    float m[1] = {-INFINITY}, lsum[1] = {0.f};
    // The wave's next stage: its K goes out once this one's K has been read, its
    // V once this one's V has, so one tile is in flight at any time. At least
    // NL loads follow K's when it is waited for (this stage's V), and V's (the
    // next K): vmcnt counts in order.
    for (; st < s_hi; st += NW) {
        const bool more = st + NW < s_hi;
        if (more) stage.fetch(table, p.bs_shift, last_block, (st + NW) * 64, Nk);
        wait_loads<NL>();
        fwd_stage<Pol, 1, true, true, false, true>(
            acc, m, lsum, qf, sk, sv, st * 64, qpos - l16, Nk, g, l16, p.scale_log2,
            [&]() __attribute__((always_inline)) {
                wait_lds();
                if (more) stage.load(sk, K, (st + NW) * 64, Nk, p.bs_shift, 0, p.kv_rs);
            },
            [&]() __attribute__((always_inline)) {
                if (more) {
                    wait_loads<NL>();
                } else {
                    wait_loads<0>();
                }
            });
        wait_lds();
        if (more) stage.load(sv, V, (st + NW) * 64, Nk, p.bs_shift, 0, p.kv_rs);
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
#pragma unroll
    for (int i = 0; i < XT; ++i)
        *reinterpret_cast<f32x4 *>(&sm.merge.acc[wave][l16][batch_col<Pol>(i, g)]) = batch_quad<Pol>(acc, i);
    if (g == 0) *reinterpret_cast<float2 *>(sm.merge.ml[wave][l16]) = make_float2(m[0], lw);
    __syncthreads();
    float *part = nullptr, *ml = nullptr;
    if (it.shares > 1) {
        part = batch_part<true>(p, it.slot, D);
        ml = batch_ml<true>(p, it.slot, D);
    }
    if (sm.merge.bad) {
        batch_plain<T, D, kBatchFew>(p, it, s_lo * 64, s_hi * 64, part, ml);
        return;
    }
    for (int i = tid; i < it.s.rows * (D / 4); i += 64 * NW) {
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
        if (it.shares > 1) {
            store4<float>(part + r * D + c, o, 1.0f);
            if (c == 0) *reinterpret_cast<float2 *>(ml + 2 * r) = make_float2(M, L);
        } else {
            batch_store<T>(p, it, r, D, c, o, M, L);
        }
    }
}

// ----------------------------------------------------------------- the many rows

template <class Pol>
__device__ __forceinline__ void batch_many_body(const BatchParams &p) {
    using T = typename Pol::T;
    constexpr int D = Pol::D, XT = D / 16, BK = Pol::ROWS;
    constexpr bool kLazy = sizeof(T) == 2;  // fp32 scores are summed from zero
    __shared__ __attribute__((aligned(16))) T sK[2][BK * D];
    __shared__ __attribute__((aligned(16))) T sV[2][BK * D];
    __shared__ int flags[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    BatchItem it;
    if (!find_item<false, false>(p, blockIdx.x, it)) return;
    const T *K = static_cast<const T *>(p.k) + it.head * D, *V = static_cast<const T *>(p.v) + it.head * D;
    const int *table = p.table + (long long)it.seq * p.table_stride;
    const unsigned last_block = p.n_blocks - 1;

    const int r0 = it.unit * kBatchMany;
    const int r = r0 + wave * 16 + l16, row = min(r, it.s.rows - 1);
    const int qpos = it.s.pos + row / p.group;
    // positions of the unit's first and last row, and of the wave's last
    const int pos_lo = it.s.pos + r0 / p.group;
    const int pos_hi = it.s.pos + min(r0 + kBatchMany - 1, it.s.rows - 1) / p.group;
    const int pos_w = it.s.pos + min(r0 + wave * 16 + 15, it.s.rows - 1) / p.group;
    typename Pol::Frag qf[1][Pol::NC];
    row_frags<Pol>(qf[0], static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D), g);
    f32x4 acc[XT][1];
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) acc[xt][0] = zero4();
    float m[1] = {-INFINITY}, lsum[1] = {0.f};

    const int Nk = min(it.s.keys, max(pos_hi + 1, 0)), n = (Nk + BK - 1) / BK;
    const int s_lo = (int)((long long)it.share * n / it.shares), s_hi = (int)((long long)(it.share + 1) * n / it.shares);
    BatchStage<Pol, 256> stage(tid);
    auto stage_next = [&](T *sk, T *sv, int st) __attribute__((always_inline)) {
        stage.load(sk, K, st * BK, Nk, p.bs_shift, wave, p.kv_rs);
        stage.load(sv, V, st * BK, Nk, p.bs_shift, wave, p.kv_rs);
        if (st + 1 < s_hi) stage.fetch(table, p.bs_shift, last_block, (st + 1) * BK, Nk);
    };
    if (s_lo < s_hi) {
        stage.fetch(table, p.bs_shift, last_block, s_lo * BK, Nk);
        stage_next(sK[0], sV[0], s_lo);
    }
    wait_stage();
    __syncthreads();
    // stages before `whole` hold no key that a row of the unit does not see
    const int whole = min(s_hi, min(Nk, pos_lo + 1) / BK);
    for (int st = s_lo; st < s_hi; ++st) {
        const int cur = (st - s_lo) & 1;
        if (st + 1 < s_hi) stage_next(sK[cur ^ 1], sV[cur ^ 1], st + 1);
        const int k0 = st * BK;
        if (k0 <= pos_w && r0 + wave * 16 < it.s.rows) {  // else no row of the wave sees the stage
            if (st < whole) {
                if (st == s_lo || !kLazy) {
                    fwd_stage<Pol, 1, true, false>(acc, m, lsum, qf, sK[cur], sV[cur], k0, qpos - l16, Nk, g, l16,
                                                   p.scale_log2);
                } else if constexpr (kLazy) {
                    fwd_stage_lazy<Pol, 1, true, false>(acc, m, lsum, qf, sK[cur], sV[cur], k0, qpos - l16, Nk, g,
                                                        l16, p.scale_log2);
                }
            } else {
                fwd_stage<Pol, 1, true, true, false, true>(acc, m, lsum, qf, sK[cur], sV[cur], k0, qpos - l16, Nk, g,
                                                           l16, p.scale_log2);
            }
        }
        wait_stage();
        __syncthreads();
    }
    const float ltot = xg_sum(lsum[0]);
    float z = 0.f * ltot;
#pragma unroll
    for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt][0]);
    float *part = nullptr, *ml = nullptr;
    if (it.shares > 1) {
        part = batch_part<false>(p, it.slot, D);
        ml = batch_ml<false>(p, it.slot, D);
    }
    const bool bad = __builtin_amdgcn_ballot_w64(z != 0.f) != 0;
    if (lane == 0) flags[wave] = bad;
    __syncthreads();
    if (flags[0] | flags[1] | flags[2] | flags[3]) {
        batch_plain<T, D, kBatchMany>(p, it, s_lo * BK, s_hi * BK, part, ml);
        return;
    }
    if (it.shares > 1) {
        const int rl = wave * 16 + l16;
        if (r < it.s.rows) {
#pragma unroll
            for (int i = 0; i < XT; ++i)
                store4<float>(part + rl * D + batch_col<Pol>(i, g), batch_quad<Pol>(acc, i), 1.0f);
            if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * rl) = make_float2(m[0], ltot);
        }
        return;
    }
    const float inv = ltot > 0.f ? 1.0f / ltot : 0.f;
    T *O = static_cast<T *>(p.o) + batch_elem(p, it, row, p.o_rs, D);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int xt = 0; xt < XT; xt += 2)
            store8_pair_bf16(O, 16 * xt, g, acc[xt][0], acc[xt + 1][0], inv, r < it.s.rows);
    } else if (r < it.s.rows) {
#pragma unroll
        for (int i = 0; i < XT; ++i) store4<T>(O + batch_col<Pol>(i, g), batch_quad<Pol>(acc, i), inv);
    }
    if (p.lse != nullptr && r < it.s.rows && g == 0)
        p.lse[batch_lse(p, it, r)] = ltot > 0.f ? (m[0] + fast_log2(ltot)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------------- the join

// The shares of a split unit: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
// D / 4 threads have a row, four elements each; where the unit has few rows
// several such groups take turns over a row's shares and meet in LDS.
template <class T, int D, bool FEW>
__device__ __forceinline__ void batch_join_body(const BatchParams &p, int w) {
    constexpr int C = D / 4, NG = 256 / C, ROWS = batch_rows<FEW>();
    __shared__ __attribute__((aligned(16))) f32x4 so[NG][C];
    BatchItem it;
    if (!find_item<FEW, true>(p, w, it)) return;
    const int tid = threadIdx.x, c = tid % C, grp = tid / C;
    const int nrows = min(ROWS, it.s.rows - it.unit * ROWS), S = it.shares;
    int together = 1;  // groups to a row
    while (together * 2 * nrows <= NG) together *= 2;
    const int turn = grp % together;
    const float *part = batch_part<FEW>(p, it.slot, D);
    const float *ml = batch_ml<FEW>(p, it.slot, D);
    const size_t pstep = (size_t)p.Hkv * ROWS * D, mstep = (size_t)p.Hkv * ROWS * 2;
    for (int r0 = 0; r0 < nrows; r0 += NG / together) {
        const int r = r0 + grp / together;
        const bool have = r < nrows;
        float M = -INFINITY, L = 0.f;
        f32x4 o = zero4();
        if (have) {
            for (int s = c; s < S; s += C) M = fmaxf(M, ml[s * mstep + 2 * r]);
        }
#pragma unroll
        for (int k = C / 2; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor(M, k, 64));
        const float mref = M == -INFINITY ? 0.f : M;
        if (have) {
            for (int s = c; s < S; s += C) {
                const float2 v = *reinterpret_cast<const float2 *>(ml + s * mstep + 2 * r);
                L += fast_exp2(v.x - mref) * v.y;
            }
#pragma unroll 4
            for (int s = turn; s < S; s += together)
                o += *reinterpret_cast<const f32x4 *>(part + s * pstep + r * D + 4 * c) *
                     fast_exp2(ml[s * mstep + 2 * r] - mref);
        }
#pragma unroll
        for (int k = C / 2; k > 0; k >>= 1) L += __shfl_xor(L, k, 64);
        if (together > 1) {
            __syncthreads();
            so[grp][c] = o;
            __syncthreads();
            if (turn == 0) {
                for (int k = 1; k < together; ++k) o += so[grp + k][c];
            }
        }
        if (have && turn == 0) batch_store<T>(p, it, it.unit * ROWS + r, D, 4 * c, o, M, L);
    }
}

// Grid: the split units the few-row form may have, then the many-row form's.
template <class T, int D>
__device__ __forceinline__ void batch_join(const BatchParams &p, int few_groups) {
    const int w = blockIdx.x;
    if (w < few_groups) {
        batch_join_body<T, D, true>(p, w);
    } else {
        batch_join_body<T, D, false>(p, w - few_groups);
    }
}

#if defined(__HIP_DEVICE_COMPILE__)
#define MXFA_BATCH(SUFFIX, POL, NW, WPS)                                                              \
    extern "C" __global__ __launch_bounds__(64 * NW) void mxfa_batch_##SUFFIX##_few(BatchParams p) {  \
        batch_few_body<POL, NW>(p);                                                                   \
    }                                                                                                 \
    extern "C" __global__ __launch_bounds__(256, WPS) void mxfa_batch_##SUFFIX##_many(BatchParams p) { \
        batch_many_body<POL>(p);                                                                      \
    }                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxfa_batch_##SUFFIX##_join(BatchParams p, int few_groups) { \
        batch_join<POL::T, POL::D>(p, few_groups);                                                    \
    }
MXFA_BATCH(b64, PolBF16<64>, 8, 3)
MXFA_BATCH(b128, PolBF16<128>, 4, 2)
MXFA_BATCH(f64, PolF32, 4, 2)
#undef MXFA_BATCH
#endif

// Items the work is cut into, about: the few-row form's work-groups have a CU
// each, so that four rounds of them even out sequences of different lengths;
// the many-row form's are resident two or three to a CU.
static int batch_target(bool few, int dtype_bf16, int d) {
    return few ? 1024 : 256 * (dtype_bf16 && d == 64 ? 3 : 2);
}

// Which forms a call launches, by what the host knows: the few-row form alone
// where no sequence can have more rows; the many-row form alone where one
// sequence has the rows; else both, each taking its own sequences.
static int batch_few_rows(const BatchParams &p) {
    const bool may_exceed = (long long)p.max_q * p.group > kBatchFew;
    return may_exceed && p.n_seq == 1 ? 0 : kBatchFew;
}
static bool batch_may_be_many(const BatchParams &p) {
    return (long long)std::min(p.max_q, p.n_tok) * p.group > kBatchFew || p.few_rows == 0;
}

// Units there can be: for the few-row form one per sequence and KV head; the
// many-row form's hold 64 rows but for a sequence's last.
static long long batch_units(const BatchParams &p, bool few) {
    if (few) return (long long)std::min(p.n_seq, p.n_tok) * p.Hkv;
    return ((long long)p.n_tok * p.group / kBatchMany + std::min(p.n_seq, p.n_tok)) * p.Hkv;
}

size_t batch_workspace_bytes(const BatchParams &q, int dtype_bf16) {
    BatchParams p = q;
    p.few_rows = batch_few_rows(p);
    size_t n = 0;
    if (p.few_rows > 0) n += batch_part_floats(batch_target(true, dtype_bf16, p.d), kBatchFew, p.d);
    if (batch_may_be_many(p)) n += batch_part_floats(batch_target(false, dtype_bf16, p.d), kBatchMany, p.d);
    return n * sizeof(float);
}

long long batch_groups(const BatchParams &q, int dtype_bf16) {
    return std::max(batch_units(q, true) + batch_target(true, dtype_bf16, q.d),
                    batch_units(q, false) + batch_target(false, dtype_bf16, q.d));
}

hipError_t launch_batch(BatchParams p, int dtype_bf16, void *workspace, hipStream_t stream) {
    static constexpr KernelId ids[3][3] = {
        {k_mxfa_batch_b64_few, k_mxfa_batch_b64_many, k_mxfa_batch_b64_join},
        {k_mxfa_batch_b128_few, k_mxfa_batch_b128_many, k_mxfa_batch_b128_join},
        {k_mxfa_batch_f64_few, k_mxfa_batch_f64_many, k_mxfa_batch_f64_join}};
    const KernelId *id = ids[!dtype_bf16 ? 2 : p.d == 128 ? 1 : 0];
    p.few_rows = batch_few_rows(p);
    const bool few = p.few_rows > 0, many = batch_may_be_many(p);
    p.target[0] = batch_target(true, dtype_bf16, p.d);
    p.target[1] = batch_target(false, dtype_bf16, p.d);
    p.part[0] = static_cast<float *>(workspace);
    p.part[1] = p.part[0] + (few ? batch_part_floats(p.target[0], kBatchFew, p.d) : 0);
    void *args[] = {&p};
    hipError_t e = hipSuccess;
    if (many)
        e = launch_kernel(id[1], dim3((unsigned)(batch_units(p, false) + p.target[1])), dim3(256), args, stream);
    if (e == hipSuccess && few)
        e = launch_kernel(id[0], dim3((unsigned)(batch_units(p, true) + p.target[0])),
                          dim3(dtype_bf16 && p.d == 64 ? 512 : 256), args, stream);
    if (e != hipSuccess) return e;
    // a split unit has two shares at least
    int few_groups = few ? (int)std::min<long long>(batch_units(p, true), p.target[0]) : 0;
    const int many_groups = many ? (int)std::min<long long>(batch_units(p, false), p.target[1]) : 0;
    void *jargs[] = {&p, &few_groups};
    return launch_kernel(id[2], dim3(few_groups + many_groups), dim3(256), jargs, stream);
}

}  // namespace mxfa
