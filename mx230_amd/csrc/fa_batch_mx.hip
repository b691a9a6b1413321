// Attention of a batch over a paged cache in 8 or 4 bits (fa_mx.h): the work of
// fa_batch.hip, whose parts, units, shares and joins these kernels share, with K and
// V made bf16 on their way to the matrix products, exactly. bf16 operands of Q and
// p are as there; in fp32 Q and p are three bf16 parts (Split3), and a product
// is three of the matrix instruction's, not six, since K and V are whole in one.
//
//   * few rows: codes and E go to LDS as they lie in the cache (a wave's own tiles, by
//     direct loads); a lane takes a quarter of a key's row, 16 bytes at d = 128 and 4
//     bits, as its share of the contraction over d, so K is converted in registers,
//     E's power in the same instruction. V is read from LDS transposed, still as
//     codes (ds_read_b64_tr_b4 / _b8): a lane has 16 keys of one column, whose powers
//     differ, so these multiply p.
//   * many rows: a thread loads a part of a key's row a stage ahead and converts it
//     once for the work-group, into the bf16 tiles of fa_batch.hip's products.
//
// Measured (us, as in fa_batch.hip; in brackets the ordinary cache, bf16 or fp32):
//   few:  64 sequences of one token, 2000-16384 long, 32/8 heads, d = 128: in 8 bits
//         195 and the join 5 (1.11 GB, 5.7 TB/s), in 4 bits 107 and 5 (0.57 GB, 5.4
//         TB/s, in pieces of 1 KB and 64 bytes) [391 and 6]; d = 64 120 and 77 in all
//         [248]; fp32 43 and 40 [125]; 512 sequences of 900, d = 128 186 and 128 in all;
//         24 sequences of 1 to 4 tokens, to 8192 long, d = 128, 8 bits: 46 and 5;
//   many: the last 2048 tokens of 32768, 32/8 heads, d = 128, 4 bits: 955 [950]; 1000
//         to 4000 tokens of short contexts 10 to 18% more than the ordinary cache: the
//         conversions and addresses, some 60 instructions a stage beside the softmax's
//         260, share the vector unit with it; fp32, 2000 tokens of 14/2 heads 39 [56];
//   both: 28 single tokens and 4 chunks of up to 512, to 8192 long, 14/2 heads, d = 64,
//         8 bits: 60 with the join [61]; fp32, 4 bits, 6 tokens and 2 chunks: 54 [57].
#include "fa_batch_items.h"
#include "fa_launch.h"
#include "fa_mx.h"

namespace mxfa {

#if defined(__HIP_DEVICE_COMPILE__)

template <int BITS_, int D_>
struct Mx {
    static constexpr int BITS = BITS_, D = D_;
    static constexpr int CB = mx_code_bytes(D, BITS), SB = mx_scale_bytes(D);  // bytes of a head's row
    static constexpr int QB = CB / 4, CH = CB / 16;  // of a quarter of it; 16-byte chunks
    static constexpr int TILE = 64 * CB;
};

// The byte offsets of positions' codes in a pool; blocks as in BatchRows.
template <class F>
struct MxRows {
    BatchRows rows;
    unsigned stride;
    MxHead head;
    __device__ __forceinline__ MxRows(const BatchParams &p, const BatchItem &it, int keys)
        : rows{p.table + (long long)it.seq * p.table_stride, p.bs_shift, keys, (unsigned)(p.n_blocks - 1)},
          stride((unsigned)p.kv_rs), head(mx_head(p, it.head)) {}
    __device__ __forceinline__ unsigned inside(int t) const {
        return (unsigned)min(t, rows.keys - 1) & ((1u << rows.shift) - 1u);
    }
    __device__ __forceinline__ size_t block(int blk) const { return (size_t)min((unsigned)blk, rows.last) * stride; }
    __device__ __forceinline__ size_t codes(int blk, int t) const { return block(blk) + head.codes + inside(t) * F::CB; }
    __device__ __forceinline__ size_t scales(int blk, int t) const { return block(blk) + head.scales + inside(t) * F::SB; }
};

// For batch_plain: elements c .. c + D / 4 - 1, a quarter of a row, of one group.
template <class F>
struct MxPlainRows {
    static constexpr int E = F::D / 4;
    MxRows<F> rows;
    const char *k, *v;
    int quarter;
    __device__ __forceinline__ MxPlainRows(const BatchParams &p, const BatchItem &it, int c)
        : rows(p, it, INT_MAX), k(static_cast<const char *>(p.k)), v(static_cast<const char *>(p.v)), quarter(c / E) {}
    size_t codes, scales;
    __device__ __forceinline__ void at(int t) {
        const int blk = rows.rows.table[t >> rows.rows.shift];
        codes = rows.codes(blk, t);
        scales = rows.scales(blk, t);
    }
    __device__ __forceinline__ void read(const char *x, float (&f)[E]) const {
        uint32_t w[F::QB / 4];
        load_words(w, x + codes + quarter * F::QB);
        const float power = mx_power((unsigned char)x[scales + quarter * E / kMxGroup]);
#pragma unroll
        for (int i = 0; i < E / 8; ++i) {
            const bf16x8 y = mx_values<F::BITS>(w + i * (F::BITS / 4), power);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[8 * i + e] = (float)y[e];
        }
    }
    __device__ __forceinline__ void read_k(float (&f)[E]) const { read(k, f); }
    __device__ __forceinline__ void read_v(float (&f)[E]) const { read(v, f); }
};

// A product's operand in registers, c + a b, and p times the powers of V's keys, for
// bf16 and (three parts) fp32.
//
// bf16: the powers multiply p after it is rounded, by adding to its exponent, two
// keys at a time: p + (E + kMxUp - 127 << 7) in 16 bits, 0 where that is negative. The
// sums are held 2^kMxUp times their size (kDown): what is left out is then less than
// 2^-126 2^-kMxUp times a code, 2^9 at most, and so less than 2^-126 in all over the 2^31
// keys that there can be. (Without that, weights below 2^-9 of the running maximum were lost
// with V near 2^-112.) p = 0 has no exponent to add to: 2^-126 is taken from every p, which
// makes a 0 the lowest integer, and so 0 with any power (whole calls in us, without, so,
// and with a branch for where some p is 0: 64 sequences of 2000-16384, d = 128, 8 bits 201.6,
// 201.5, 205.8, d = 64, 4 bits 75.0, 75.3, 77.4; 512 of 900, d = 128, 4 bits 127.6, 128.6,
// 129.9). In stages that hold a key that a row does
// not see all multiply in fp32. With E up to kMxMost no exponent passes 254 - 8 (p is at
// most kLazySum); a piece that met a larger one (V above 2^63, or NaN) or whose sums
// overflow runs in plain arithmetic.
constexpr unsigned kMxMost = 190, kMxUp = 40;
template <class T>
struct MxOperand;
template <>
struct MxOperand<u16> {
    using B = bf16x8;
    using Power = u16;
    static constexpr float kDown = 0x1p-40f;
    static_assert(kDown * (float)(1ull << kMxUp) == 1.0f && 16 + kMxMost + kMxUp < 255);
    struct Packed {
        u32x4 w[2];  // keys 2 i, 2 i + 1 in word i
    };
    // EXACT: the power itself in bf16
    template <bool EXACT>
    __device__ static __forceinline__ Power power(unsigned E) { return (u16)((E + kMxUp - (EXACT ? 0 : 127)) << 7); }
    __device__ static __forceinline__ f32x4 mma(bf16x8 a, const B &b, f32x4 c) { return PolBF16<64>::mma(a, b, c); }
    __device__ static __forceinline__ Packed prepare(const f32x4 (&p)[4]) {
        const float least = 0x1p-126f;
        return Packed{{__builtin_bit_cast(u32x4, PolBF16<64>::pack(p[0] - least, p[1] - least)),
                       __builtin_bit_cast(u32x4, PolBF16<64>::pack(p[2] - least, p[3] - least))}};
    }
    template <bool EXACT>
    __device__ static __forceinline__ void scaled(B (&f)[2], const Packed &pk, const f32x4 (&p)[4], const Power *power) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 e = *reinterpret_cast<const u32x4 *>(power + 8 * h);
            if constexpr (EXACT) {
                f32x4 x[2];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i / 4][i % 4] = p[2 * h + i / 4][i % 4] * __uint_as_float(i & 1 ? e[i / 2] & 0xffff0000u : e[i / 2] << 16);
                f[h] = PolBF16<64>::pack(x[0], x[1]);
            } else {
                u32x4 r;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a = pk.w[h][i], b = e[i];
                    const i16x2 x = __builtin_elementwise_add_sat(__builtin_bit_cast(i16x2, a), __builtin_bit_cast(i16x2, b));
                    r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, i16x2{0, 0}));
                }
                f[h] = __builtin_bit_cast(B, r);
            }
        }
    }
};
template <>
struct MxOperand<float> {
    using B = Split3;
    using Power = float;
    // p times a power of down to 2^-117 keeps its parts (kPartMin)
    static constexpr float kDown = kPartDown;
    struct Packed {};
    template <bool>
    __device__ static __forceinline__ Power power(unsigned E) { return mx_power(E); }
    __device__ static __forceinline__ f32x4 mma(bf16x8 a, const B &b, f32x4 c) {
        c = PolBF16<64>::mma(a, b.l, c);
        c = PolBF16<64>::mma(a, b.m, c);
        return PolBF16<64>::mma(a, b.h, c);
    }
    __device__ static __forceinline__ Packed prepare(const f32x4 (&)[4]) { return Packed{}; }
    template <bool EXACT>
    __device__ static __forceinline__ void scaled(B (&f)[2], const Packed &, const f32x4 (&p)[4], const Power *power) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 *e = reinterpret_cast<const f32x4 *>(power + 8 * h);
            f[h] = split3(p[2 * h] * kPartUp * e[0], p[2 * h + 1] * kPartUp * e[1]);
        }
    }
};

// A lane's D / 4 elements of a row of Q, quarter g, in the order of K's codes. True
// for the wave where a row's parts are not 24 bits (fp32: as split_row).
template <class F, class T>
__device__ __forceinline__ bool mx_row(typename MxOperand<T>::B (&f)[F::D / 32], const T *row, int g) {
    row += g * (F::D / 4);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int c = 0; c < F::D / 32; ++c) f[c] = *reinterpret_cast<const bf16x8 *>(row + 8 * c);
        return false;
    } else {
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < F::D / 32; ++c) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(row + 8 * c), b = *reinterpret_cast<const f32x4 *>(row + 8 * c + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(a[e]), fabsf(b[e])));
            f[c] = split3(a, b);
        }
        uint64_t some = __builtin_amdgcn_ballot_w64(mx > 0.f), enough = __builtin_amdgcn_ballot_w64(mx >= kPartMin);
        some |= some >> 32;
        enough |= enough >> 32;
        return (((some | some >> 16) & ~(enough | enough >> 16)) & 0xffff) != 0;
    }
}

// Waits for Q's loads. The compiler knows of no others, and where a use may be the first
// after them it waits until none of any kind is left: without this in every stage (the
// kernel in us at the step that brought it, 64 sequences of 2000-16384, 32/8 heads, d = 128, 4
// bits: 121 and 110; since Q comes a piece ahead, whole calls: 512 sequences of 900, 8 bits,
// 190 and 185, others the same).
template <class T, int N>
__device__ __forceinline__ void mx_arrived(typename MxOperand<T>::B (&f)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if constexpr (sizeof(T) == 2) {
            asm volatile("" : "+v"(f[c]));
        } else {
            asm volatile("" : "+v"(f[c].h), "+v"(f[c].m), "+v"(f[c].l));
        }
    }
}

// ------------------------------------------------------------------ the few rows

// V's tiles, and where the waves meet at a piece's end: in the same LDS, or apart where a
// work-group sends for the next piece before and has a CU's LDS to itself.
template <class Values, class Merge>
union MxFewShared {
    Values values;
    Merge merge;
};
template <class Values, class Merge>
struct MxFewApart {
    Values values;
    alignas(16) Merge merge;
};
template <class F, class T, int NW, bool AHEAD>
struct MxFewSmem {
    struct Keys {
        char k[F::TILE];
        uint32_t e[64];             // E of a key in its low SB bytes
        int blk[2][64], first[64];  // blocks of its stages; of the next piece's first
    };
    struct Values {
        char v[NW][F::TILE];
        uint32_t e[NW][64];
        typename MxOperand<T>::Power power[NW][F::SB][64];
    };
    using Merge = BatchFewMerge<F::D, NW>;
    static constexpr bool APART = AHEAD && NW * sizeof(Keys) + sizeof(Values) + sizeof(Merge) + 16 <= 160 * 1024;
    Keys keys[NW];
    std::conditional_t<APART, MxFewApart<Values, Merge>, MxFewShared<Values, Merge>> end;
};

// Codes in LDS: chunk c of row r at slot c ^ kswz(r) (K) or c ^ vswz(r) (V).
template <class F>
__device__ __forceinline__ int mx_kswz(int r) {
    // a score operand reads rows that differ in bits 0, 1, 4, 5, one quarter at a time
    return F::CH == 8 ? (((r >> 1) & 1) | ((r >> 4) & 3) << 1) : F::CH == 4 ? (r >> 4) & 3 : (r >> 4) & 1;
}
template <class F>
__device__ __forceinline__ int mx_vswz(int r) {
    // a transposing read: rows that differ in their low bits
    return F::CH == 8 ? (((r >> 1) & 3) | ((r >> 4) & 1) << 2) : F::CH == 4 ? (r >> 2) & 3 : (r >> 3) & 1;
}

// A wave's loads of a stage's codes, CH of 64 chunks, and E. A load's 64 / CH rows
// lie in a run where blocks are as large (`runs`): its address is then a uniform one
// and the lane's constant. The stage that ends the sequence goes by each row's
// own, the last one's past it: what lies behind a sequence is not read.
template <class F>
struct MxStage {
    static constexpr int LOADS = F::CH + 1, ROWS = 64 / F::CH;
    template <class Swz>
    __device__ static __forceinline__ void load(char *tile, uint32_t *es, const char *X, const MxRows<F> &rows, const int *blk,
                                                int k0, int lane, bool runs, Swz swz) {
        const uint32_t base = lds_addr(tile);
        const int mine = blk[lane];
        if (runs && k0 + 64 <= rows.rows.keys) {
#pragma unroll
            for (int k = 0; k < F::CH; ++k) {
                const int row = k * ROWS + lane / F::CH;
                const char *at = X + rows.codes(__builtin_amdgcn_readlane(mine, k * ROWS), k0 + k * ROWS);
                lds_dma16_u(base + k * 1024, at, (uint32_t)((lane / F::CH) * F::CB + (((lane % F::CH) ^ swz(row)) << 4)));
            }
        } else {
#pragma unroll
            for (int k = 0; k < F::CH; ++k) {
                const int row = k * ROWS + lane / F::CH, c = (lane % F::CH) ^ swz(row);
                lds_dma16(base + k * 1024, X + rows.codes(blk[row], k0 + row) + 16 * c);
            }
        }
        const char *e = X + rows.scales(mine, k0 + lane);
        if constexpr (F::SB == 4) {
            lds_dma4(lds_addr(es), e);
        } else {
            lds_dma2(lds_addr(es), e);
        }
    }
};

// One 64-key stage: key 16 a + 4 t + b of it is row 4 a + b of score tile t, so a lane
// (g, l16) holds the scores of keys 16 g .. 16 g + 15 of row l16, in order: the 16
// keys whose codes a transposing read of V brings it. p is relative to the running
// m, which rises only where a lane's sum of p passes kLazySum (fwd_stage_lazy's
// reasons), at the wave's FIRST stage, or while m is -infinity for some row: where every
// score so far overflowed to that, the next may be finite and yet so low that p relative to
// 0 is 0. most: the largest E of V so far.
template <class F, class T, bool FIRST, bool MASK, class AfterK, class BeforeV>
__device__ __forceinline__ void mx_few_stage(f32x4 (&acc)[F::D / 16], float &m, float &lsum, unsigned &most,
                                             const typename MxOperand<T>::B (&qf)[F::D / 32], const char *sk,
                                             const uint32_t *ke, const char *sv, const uint32_t *ve,
                                             typename MxOperand<T>::Power (*vp)[64], int lim, int lane, float xmul,
                                             AfterK after_k, BeforeV before_v) {
    using Op = MxOperand<T>;
    constexpr int NC = F::D / 32, XT = F::D / 16;
    const int g = lane >> 4, l16 = lane & 15;
    f32x4 s[4], pv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int row = 16 * (l16 >> 2) + 4 * t + (l16 & 3);
        uint32_t w[F::QB / 4];
        if constexpr (F::QB >= 16) {
#pragma unroll
            for (int i = 0; i < F::QB / 16; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(sk + row * F::CB + (((F::QB / 16 * g + i) ^ mx_kswz<F>(row)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = x[e];
            }
        } else {  // (half a chunk)
            const u32x2 x = *reinterpret_cast<const u32x2 *>(sk + row * F::CB + (((g >> 1) ^ mx_kswz<F>(row)) << 4) + 8 * (g & 1));
            w[0] = x[0];
            w[1] = x[1];
        }
        const float power = mx_power(reinterpret_cast<const unsigned char *>(ke + row)[g * F::SB / 4]);
        f32x4 c = zero4();
#pragma unroll
        for (int i = 0; i < NC; ++i) c = Op::mma(mx_values<F::BITS>(w + i * (F::BITS / 4), power), qf[i], c);
        s[t] = c;
    }
    after_k();
    if constexpr (MASK) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = 4 * t + r > lim ? -INFINITY : s[t][r];
        }
    }
    auto exps = [&](float sub) __attribute__((always_inline)) {
        float ls = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pv[t][r] = fast_exp2(__builtin_fmaf(s[t][r], xmul, -sub));
                ls += pv[t][r];
            }
        }
        return ls;
    };
    auto raise = [&]() __attribute__((always_inline)) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[t][r]);
        }
        mx = fmaxf(xg_max(mx) * xmul, m);
        const float to = mx == -INFINITY ? 0.f : mx;  // (a row that sees no key)
        if constexpr (!FIRST) {
            const float corr = fast_exp2(m - to);
            lsum *= corr;
#pragma unroll
            for (int xt = 0; xt < XT; ++xt) acc[xt] *= corr;
        }
        m = mx;
        lsum += exps(to);
    };
    if constexpr (FIRST) {
        raise();
    } else {
        const bool none = m == -INFINITY;  // no key seen, or every score so far -infinity
        const float ls = exps(none ? 0.f : m);
        if (__builtin_amdgcn_ballot_w64(none || ls > kLazySum) != 0) {
            raise();
        } else {
            lsum += ls;
        }
    }
    before_v();
    // the powers of V's keys, a lane a key
    const uint32_t e = ve[lane];
#pragma unroll
    for (int grp = 0; grp < F::SB; ++grp) {
        const unsigned E = (e >> (8 * grp)) & 255u;
        most = max(most, E);
        vp[grp][lane] = Op::template power<MASK>(E);
    }
    wait_lds();
    typename Op::Packed pk;
    if constexpr (!MASK) pk = Op::prepare(pv);
#pragma unroll
    for (int grp = 0; grp < F::SB; ++grp) {
        typename Op::B pf[2];
        Op::template scaled<MASK>(pf, pk, pv, vp[grp] + 16 * g);
#pragma unroll
        for (int xt = 2 * grp; xt < 2 * grp + 2; ++xt) {
            uint32_t w[F::BITS / 2];  // 16 keys of column 16 xt + l16
            if constexpr (F::BITS == 4) {
                const int row = 16 * g + l16;
                const i32x2 x = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                    (lds_i32x2 *)(sv + row * F::CB + (((xt >> 1) ^ mx_vswz<F>(row)) << 4) + 8 * (xt & 1)));
                w[0] = x[0];
                w[1] = x[1];
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = 16 * g + 8 * h + (l16 >> 1);
                    const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (lds_i32x2 *)(sv + row * F::CB + ((xt ^ mx_vswz<F>(row)) << 4) + 8 * (l16 & 1)));
                    w[2 * h] = x[0];
                    w[2 * h + 1] = x[1];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[xt] = Op::mma(mx_values<F::BITS>(w + h * (F::BITS / 4), 1.0f), pf[h], acc[xt]);
        }
    }
}

// Which of the form's `n` work-groups a block of a launch of its own is: each XCD (blocks 8
// apart) has them one after another, so the heads of a run, whose E share lines, share
// an L2: 610 MB read and 574 (4 bits, d = 128), which is what it needs. us, 64
// sequences of 2000-16384, 32/8 heads, in order and so: d = 128, 4 bits 109 and 107,
// 8 bits 198 and 195; d = 64 79.6 and 78, 122.7 and 120.8. Beside the many-row form, where they
// would crowd some XCDs, in order (fp32, 6 tokens and 2 chunks: 30.6 us and 38.5).
__device__ __forceinline__ int mx_few_group(int block, int n) {
    const int xcd = block & 7, each = n >> 3, more = n & 7;
    return xcd * each + min(xcd, more) + (block >> 3);
}

// A work-group's run of pieces, as batch_few_piece: their loads and waits. AHEAD: a wave
// that is done with a piece sends for its first stage of the next one before the waves
// meet, V only where its tiles are not what they meet in (APART); Q has come a piece
// ahead. us, without and with it: 512 sequences of 900 tokens, 32/8 heads, d = 128, 8 bits
// 204 and 186, 4 bits 150 and 128 (V after they met: 135); 64 of 2000-16384, 4 bits
// 110 and 107; one of 4096, which has no next piece, 7.0 and 7.7: a batch of one does
// without (`one`), and beside the many-row form's registers it brought nothing.
template <class F, class T, int NW, bool AHEAD>
__device__ __forceinline__ void mx_few_body(const BatchParams &p, int group, MxFewSmem<F, T, NW, AHEAD> &sm) {
    using Stage = MxStage<F>;
    constexpr int D = F::D, XT = D / 16, ROWS = kBatchFew, NL = Stage::LOADS;
    constexpr bool APART = MxFewSmem<F, T, NW, AHEAD>::APART;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const char *K = static_cast<const char *>(p.k), *V = static_cast<const char *>(p.v);
    const bool runs = (1 << p.bs_shift) >= Stage::ROWS;
    auto &t = sm.keys[wave];
    auto &values = sm.end.values;

    // the blocks of stage `st` of a piece that ends before stage `hi`
    auto fetch = [&](int *to, const BatchItem &of, int st, int hi) __attribute__((always_inline)) {
        const MxRows<F> rows(p, of, of.s.keys);
        lds_dma4(lds_addr(to), rows.rows.table + rows.rows.block_at(min(st, hi - 1) * 64 + lane));
    };
    auto load_k = [&](const BatchItem &of, int st, const int *blk) __attribute__((always_inline)) {
        Stage::load(t.k, t.e, K, MxRows<F>(p, of, of.s.keys), blk, st * 64, lane, runs, mx_kswz<F>);
    };
    auto load_v = [&](const BatchItem &of, int st, const int *blk) __attribute__((always_inline)) {
        Stage::load(values.v[wave], values.e[wave], V, MxRows<F>(p, of, of.s.keys), blk, st * 64, lane, runs, mx_vswz<F>);
    };
    auto load_q = [&](typename MxOperand<T>::B (&to)[D / 32], const BatchItem &of) __attribute__((always_inline)) {
        return mx_row<F, T>(to, static_cast<const T *>(p.q) + batch_elem(p, of, min(l16, of.s.rows - 1), p.q_rs, D), g);
    };

    FewRun run(p, group);
    BatchItem it = run.item(), nx = it;
    FewPiece f, nf;
    if (!run.next(it, f)) return;
    typename MxOperand<T>::B qf[D / 32];
    bool low;
    auto begin = [&]() __attribute__((always_inline)) {
        if (f.lo + wave < f.hi) fetch(t.first, it, f.lo + wave, f.hi);
        low = load_q(qf, it);
        mx_arrived<T>(qf);
        if (f.lo + wave < f.hi) {
            wait_loads<0>();
            fetch(t.blk[1], it, f.lo + wave + NW, f.hi);
            load_k(it, f.lo + wave, t.first);
            load_v(it, f.lo + wave, t.first);
        }
    };
    if (AHEAD) begin();
    for (;;) {
        if (!AHEAD) begin();
        const bool other = AHEAD && run.next(nx, nf), ahead = other && nf.lo + wave < nf.hi;
        const int s_hi = f.hi, Nk = it.s.keys;
        int st = f.lo + wave, n = 0;
        const int qpos = it.s.pos + min(l16, it.s.rows - 1) / p.group;
        f32x4 acc[XT];
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) acc[xt] = zero4();
        float m = -INFINITY, lsum = 0.f;
        unsigned most = 0;
        // stages before `whole` hold no key that a row does not see
        const int whole = min(Nk, it.s.pos + 1) / 64;
        // what the next piece begins with
        typename MxOperand<T>::B qn[D / 32];
        bool lown = false;
        auto next_up = [&]() __attribute__((always_inline)) {
            if (ahead) fetch(t.first, nx, nf.lo + wave, nf.hi);
            if (other) lown = load_q(qn, nx);
        };
        // The wave's next stage: its K goes out once this one's K has been read, with the
        // blocks of the stage after it, and its V once this one's V has; the blocks of the n-th
        // are in blk[n & 1], of the first in `first`. vmcnt counts in order: NL loads (this stage's
        // V) follow K, NL + 1 (the blocks and the next K) follow V;
        // what else goes out in a piece's first stage only makes these waits longer.
        auto stage = [&](auto first, auto mask) __attribute__((always_inline)) {
            const bool more = st + NW < s_hi;
            wait_loads<NL>();
            auto after_k = [&]() __attribute__((always_inline)) {
                wait_lds();
                if (decltype(first)::value) next_up();
                if (more) {
                    fetch(t.blk[n & 1], it, st + 2 * NW, s_hi);  // (this stage's: its V is out already)
                    load_k(it, st + NW, t.blk[(n + 1) & 1]);
                }
            };
            auto before_v = [&]() __attribute__((always_inline)) {
                if (more) {
                    wait_loads<NL + 1>();
                } else {
                    wait_loads<0>();
                }
            };
            const int lim = min(qpos, Nk - 1) - st * 64 - 16 * g;
            mx_few_stage<F, T, decltype(first)::value, decltype(mask)::value>(
                acc, m, lsum, most, qf, t.k, t.e, values.v[wave], values.e[wave], values.power[wave], lim, lane, p.scale_log2,
                after_k, before_v);
            wait_lds();
            if (more) load_v(it, st + NW, t.blk[(n + 1) & 1]);
            st += NW;
            ++n;
        };
        using std::false_type;
        using std::true_type;
        if (st < s_hi) {
            stage(true_type{}, true_type{});
        } else {
            next_up();
            if constexpr (AHEAD) mx_arrived<T>(qn);
        }
        while (st < min(s_hi, whole)) stage(false_type{}, false_type{});
        while (st < s_hi) stage(false_type{}, true_type{});

        if constexpr (AHEAD) mx_arrived<T>(qn);
        if (ahead) {
            wait_loads<0>();
            fetch(t.blk[1], nx, nf.lo + wave + NW, nf.hi);
            load_k(nx, nf.lo + wave, t.first);
            if constexpr (APART) load_v(nx, nf.lo + wave, t.first);
        }
        const float lw = xg_sum(lsum);
        float z = 0.f * lw;
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt]);
        const bool bad = __builtin_amdgcn_ballot_w64(z != 0.f || most > kMxMost) != 0 || low;
        batch_few_finish<T, D, NW, 64 * NW>(
            p, it, f.slot, sm.end.merge, m, lw, bad,
            [&](int i) __attribute__((always_inline)) { return acc[i] * MxOperand<T>::kDown; },
            [&](int i) __attribute__((always_inline)) { return 16 * i + 4 * g; },
            [&](float *part, float *ml) __attribute__((always_inline)) {
                batch_plain<T, D, ROWS, MxPlainRows<F>>(p, it, 0, f.lo * 64, f.hi * 64, part, ml);
            });
        if constexpr (AHEAD) {
            if (!other) return;
            if constexpr (!APART) {
                barrier_lds();  // V's tiles are where the waves met
                if (ahead) load_v(nx, nf.lo + wave, t.first);
            }
            it = nx;
            f = nf;
            low = lown;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) qf[c] = qn[c];
        } else {
            if (!run.next(it, f)) return;
            barrier_lds();
        }
    }
}

// ----------------------------------------------------------------- the many rows

// The products' policy: K and V as bf16 tiles, Q and p in bf16 or in three parts.
template <int D_>
struct PolMxF32 : PolRows<D_> {
    using Base = PolRows<D_>;
    using Op = MxOperand<float>;
    using Frag = typename Base::Frag;
    using T = u16;
    using QFrag = Split3;
    using ChainB = Split3;
    __device__ static __forceinline__ f32x4 mma(Frag a, const QFrag &b, f32x4 c) { return Op::mma(a, b, c); }
    __device__ static __forceinline__ ChainB pack(const f32x4 &a, const f32x4 &b) { return split3(a, b); }
    __device__ static __forceinline__ f32x4 chain(f32x4 acc, const ChainB &b, const T *tile, int y0, int blk, int g, int l16) {
        return Op::mma(Base::chain_a(tile, y0, blk, g, l16), b, acc);
    }
};
template <class T, int D>
using PolMx = std::conditional_t<sizeof(T) == 2, PolRows<D>, PolMxF32<D>>;

template <int D, int NW>
struct MxManySmem {
    __attribute__((aligned(16))) u16 k[2][64 * D], v[2][64 * D];
    int bad[NW];
};

// A thread's part of a stage of K or V, of NT threads': loaded as codes, written to
// the tile as bf16.
template <class F, int NT>
struct MxPart {
    static constexpr int TPR = NT / 64, E = F::D / TPR, B = E * F::BITS / 8;  // threads of a row, elements, bytes
    uint32_t w[B / 4];
    float power;
    __device__ __forceinline__ void load(const char *codes, const char *scales) {
        load_words(w, codes);
        power = mx_power((unsigned char)*scales);
    }
    __device__ __forceinline__ void write(u16 *tile, int row, int part) const {
        char *base = reinterpret_cast<char *>(tile) + row * (2 * F::D);
#pragma unroll
        for (int i = 0; i < E / 8; ++i)
            *reinterpret_cast<bf16x8 *>(base + ((((part * E) / 8 + i) ^ PolRows<F::D>::swz(row)) << 4)) =
                mx_values<F::BITS>(w + i * (F::BITS / 4), power);
    }
};

// One unit's share, as batch_many_body, NW waves of 16 QT rows.
template <class F, class T, int QT, int NW>
__device__ __forceinline__ void mx_many_body(const BatchParams &p, int block, MxManySmem<F::D, NW> &sm) {
    using Pol = PolMx<T, F::D>;
    using Part = MxPart<F, 64 * NW>;
    constexpr int D = F::D, XT = D / 16, BK = 64, ROWS = 16 * QT * NW;
    constexpr bool kPrio = true;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    BatchItem it;
    if (!find_item<ROWS>(p, batch_order(p, block), it)) return;
    const char *K = static_cast<const char *>(p.k), *V = static_cast<const char *>(p.v);

    const int r0 = it.unit * ROWS, rw = r0 + wave * 16 * QT;  // the unit's and the wave's first row
    const int last_row = it.s.rows - 1;
    RowPos<QT> qpos;
    typename Pol::QFrag qf[QT][Pol::NC];
    bool low = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = min(rw + 16 * qt + l16, last_row);
        qpos.at[qt] = it.s.pos + row / p.group;
        const T *q = static_cast<const T *>(p.q) + batch_elem(p, it, row, p.q_rs, D);
        if constexpr (sizeof(T) == 2) {
            row_frags<Pol>(qf[qt], q, g);
        } else {
            low |= split_row(qf[qt], q, g, 1.0f, true);
        }
    }
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
    const MxRows<F> rows(p, it, Nk);
    int s_lo, s_hi;
    share_stages(it, n, s_lo, s_hi);

    // the stage after the next: its block; the next: its codes, in registers
    const int key = tid / Part::TPR, part = tid % Part::TPR;
    Part xk, xv;
    int blk = 0;
    auto fetch = [&](int st) __attribute__((always_inline)) { blk = rows.rows.table[rows.rows.block_at(st * BK + key)]; };
    auto load = [&](int st) __attribute__((always_inline)) {
        const size_t codes = rows.codes(blk, st * BK + key) + part * Part::B;
        const size_t scales = rows.scales(blk, st * BK + key) + part * Part::E / kMxGroup;
        xk.load(K + codes, K + scales);
        xv.load(V + codes, V + scales);
        if (st + 1 < s_hi) fetch(st + 1);
    };
    auto write = [&](int buf) __attribute__((always_inline)) {
        xk.write(sm.k[buf], key, part);
        xv.write(sm.v[buf], key, part);
    };
    if (s_lo < s_hi) {
        fetch(s_lo);
        load(s_lo);
        write(0);
    }
    barrier_lds();
    const int whole = min(s_hi, min(Nk, pos_lo + 1) / BK);
    const bool some = rw <= last_row;  // the wave has rows
    auto main_stage = [&](auto buf, auto first, int st) __attribute__((always_inline)) {
        constexpr int B = decltype(buf)::value;
        if (st + 1 < s_hi) load(st + 1);
        if (some) {
            if constexpr (decltype(first)::value) {
                fwd_stage<Pol, QT, true, false, kPrio>(acc, m, lsum, qf, sm.k[B], sm.v[B], st * BK, qpos, Nk, g, l16,
                                                       p.scale_log2);
            } else {
                fwd_stage_lazy<Pol, QT, true, false, kPrio>(acc, m, lsum, qf, sm.k[B], sm.v[B], st * BK, qpos, Nk, g, l16,
                                                            p.scale_log2);
            }
        }
        if (st + 1 < s_hi) write(B ^ 1);
        barrier_lds();
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
        if (st + 1 < s_hi) load(st + 1);
        if (some && st * BK <= pos_w)  // else no row of the wave sees the stage
            fwd_stage<Pol, QT, true, true, kPrio, true>(acc, m, lsum, qf, sm.k[cur], sm.v[cur], st * BK, qpos, Nk, g, l16,
                                                        p.scale_log2);
        if (st + 1 < s_hi) write(cur ^ 1);
        barrier_lds();
    }
    float ltot[QT], z = 0.f;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        ltot[qt] = xg_sum(lsum[qt]);
        z += 0.f * ltot[qt];
#pragma unroll
        for (int xt = 0; xt < XT; ++xt) z += zero_of(acc[xt][qt]);
    }
    float *ws = nullptr, *ml = nullptr;
    if (it.shares > 1) {
        ws = batch_part(p.part[1], it.slot, ROWS, D);
        ml = batch_ml(p.part[1], p.slots, it.slot, ROWS, D);
    }
    const bool bad = __builtin_amdgcn_ballot_w64(z != 0.f) != 0 || low;
    if (lane == 0) sm.bad[wave] = bad;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= sm.bad[w];
    if (any) {
        for (int i = 0; i < ROWS; i += 16 * NW)
            batch_plain<T, D, ROWS, MxPlainRows<F>>(p, it, i, s_lo * BK, s_hi * BK, ws, ml);
        return;
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = rw + 16 * qt + l16, rl = r - r0;
        const bool have = r < it.s.rows;
        if (it.shares > 1) {
            if (have) {
#pragma unroll
                for (int i = 0; i < XT; ++i) store4<float>(ws + rl * D + 16 * i + 4 * g, acc[i][qt], 1.0f);
                if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * rl) = make_float2(m[qt], ltot[qt]);
            }
            continue;
        }
        const float inv = batch_inverse(ltot[qt], qpos.at[qt]);
        T *O = static_cast<T *>(p.o) + batch_elem(p, it, min(r, last_row), p.o_rs, D);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int xt = 0; xt < XT; xt += 2)
                store8_pair_bf16(O, 16 * xt, g, acc[xt][qt], acc[xt + 1][qt], inv, have);
        } else if (have) {
#pragma unroll
            for (int xt = 0; xt < XT; ++xt) store4<float>(O + 16 * xt + 4 * g, acc[xt][qt], inv);
        }
        if (p.lse != nullptr && have && g == 0)
            p.lse[batch_lse(p, it, r)] = ltot[qt] > 0.f ? (m[qt] + fast_log2(ltot[qt])) * kLn2 : -INFINITY;
    }
}

// Both forms in one launch, as batch_both_body.
template <class F, class T, int QT, int NW>
__device__ __forceinline__ void mx_both_body(const BatchParams &p, int few_groups) {
    __shared__ __attribute__((aligned(16))) union {
        MxFewSmem<F, T, NW, false> few;
        MxManySmem<F::D, NW> many;
    } sm;
    if ((int)blockIdx.x < few_groups) {
        mx_few_body<F, T, NW, false>(p, blockIdx.x, sm.few);
    } else {
        mx_many_body<F, T, QT, NW>(p, (int)blockIdx.x - few_groups, sm.many);
    }
}

#define MXFA_BATCH_MX_FEW(NAME, BITS, D, T, AHEAD)                                                           \
    extern "C" __global__ __launch_bounds__(64 * kMxFewWaves) void mxfa_batch_##NAME(BatchParams p) {        \
        __shared__ __attribute__((aligned(16))) MxFewSmem<Mx<BITS, D>, T, kMxFewWaves, AHEAD> sm;            \
        mx_few_body<Mx<BITS, D>, T, kMxFewWaves, AHEAD>(p, mx_few_group(blockIdx.x, gridDim.x), sm);         \
    }
#define MXFA_BATCH_MX_MANY(MANY, BOTH, BITS, D, T, QT, NW, WPS, BOTH_WPS)                                    \
    extern "C" __global__ __launch_bounds__(64 * NW, WPS) void mxfa_batch_##MANY(BatchParams p) {            \
        __shared__ __attribute__((aligned(16))) MxManySmem<D, NW> sm;                                        \
        mx_many_body<Mx<BITS, D>, T, QT, NW>(p, blockIdx.x, sm);                                             \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(64 * NW, BOTH_WPS) void mxfa_batch_##BOTH(BatchParams p, int few_groups) { \
        mx_both_body<Mx<BITS, D>, T, QT, NW>(p, few_groups);                                                 \
    }
#define MXFA_BATCH_MX(BITS)                                                                                  \
    MXFA_BATCH_MX_FEW(x##BITS##b64_few, BITS, 64, u16, true)                                                 \
    MXFA_BATCH_MX_FEW(x##BITS##b64_one, BITS, 64, u16, false)                                                \
    MXFA_BATCH_MX_MANY(x##BITS##b64_many, x##BITS##b64_both, BITS, 64, u16, 2, 4, 3, 3)                      \
    MXFA_BATCH_MX_MANY(x##BITS##b64_many64, x##BITS##b64_both64, BITS, 64, u16, 1, 4, 4, 3)                  \
    MXFA_BATCH_MX_FEW(x##BITS##b128_few, BITS, 128, u16, true)                                               \
    MXFA_BATCH_MX_FEW(x##BITS##b128_one, BITS, 128, u16, false)                                              \
    MXFA_BATCH_MX_MANY(x##BITS##b128_many, x##BITS##b128_both, BITS, 128, u16, 2, 4, 2, 2)                   \
    MXFA_BATCH_MX_MANY(x##BITS##b128_many64, x##BITS##b128_both64, BITS, 128, u16, 1, 4, 2, 2)               \
    MXFA_BATCH_MX_FEW(x##BITS##f64_few, BITS, 64, float, true)                                               \
    MXFA_BATCH_MX_FEW(x##BITS##f64_one, BITS, 64, float, false)                                              \
    MXFA_BATCH_MX_MANY(x##BITS##f64_many, x##BITS##f64_both, BITS, 64, float, 1, kBatchF32Waves, 4, 4)
MXFA_BATCH_MX(8)
MXFA_BATCH_MX(4)
#undef MXFA_BATCH_MX
#undef MXFA_BATCH_MX_MANY
#undef MXFA_BATCH_MX_FEW

#endif

}  // namespace mxfa
