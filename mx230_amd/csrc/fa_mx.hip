// The write of new tokens into a microscaled cache (fa_mx.h), with rotary
// positions, and the read of its rows back.
//
// A code hangs on which side of a border its value lies. So that equal tokens get
// equal codes whatever computes them, K turns in 64 bits (angle, cosine, sine,
// products; off by some 1e-11 at positions of 10^5, a border is met that closely once in
// 10^9 values) and is rounded to 32; E and the codes, to nearest even, follow from
// those 32 bits alone. Q turns in 32 bits, as in the ordinary append.
#include <limits.h>

#include <algorithm>

#include "fa_launch.h"
#include "fa_mx.h"

namespace mxfa {

// A work-group of 256 threads has as many tokens, of U threads each, as lie whole in
// its waves: Q is turned in place where the caller wants that, and an element's
// other half is then read before the wave stores either. mx_token: the thread's
// token, past the last one for lanes that have none.
__host__ __device__ inline int mx_tokens(int U) { return 4 * (64 / U); }

#if defined(__HIP_DEVICE_COMPILE__)

// cos and sin of an angle in turns: reduced to [-1/8, 1/8], then Taylor's series,
// whose first terms left out are z^17 / 17! <= 5e-17 and z^16 / 16! <= 1.1e-15 at z =
// pi / 4. The position times the frequency over 2 pi is rounded three times, so
// the angle is off by up to 3 x 2^-53 of itself.
__device__ __forceinline__ void turn_angle64(double turns, double &c, double &s) {
    turns -= __builtin_rint(turns);
    const double quarter = __builtin_rint(4.0 * turns);
    const double z = 6.283185307179586 * __builtin_fma(-0.25, quarter, turns), w = z * z;
    const int q = (int)quarter & 3;
    double sn = -1.0 / 1307674368000.0;
    sn = __builtin_fma(w, sn, 1.0 / 6227020800.0);
    sn = __builtin_fma(w, sn, -1.0 / 39916800.0);
    sn = __builtin_fma(w, sn, 1.0 / 362880.0);
    sn = __builtin_fma(w, sn, -1.0 / 5040.0);
    sn = __builtin_fma(w, sn, 1.0 / 120.0);
    sn = __builtin_fma(w, sn, -1.0 / 6.0);
    sn = __builtin_fma(z * w, sn, z);
    double cs = -1.0 / 87178291200.0;
    cs = __builtin_fma(w, cs, 1.0 / 479001600.0);
    cs = __builtin_fma(w, cs, -1.0 / 3628800.0);
    cs = __builtin_fma(w, cs, 1.0 / 40320.0);
    cs = __builtin_fma(w, cs, -1.0 / 720.0);
    cs = __builtin_fma(w, cs, 1.0 / 24.0);
    cs = __builtin_fma(w, cs, -0.5);
    cs = __builtin_fma(w, cs, 1.0);
    const double a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
    c = q == 1 || q == 2 ? -a : a;
    s = q >= 2 ? -b : b;
}

// 8 neighbouring elements as they lie in memory, and as floats.
template <class T>
struct Raw8 {
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const u32x4 *>(p)[i];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(T) == 2) {
                x[e] = __uint_as_float(e & 1 ? w[0][e / 2] & 0xffff0000u : w[0][e / 2] << 16);
            } else {
                x[e] = __uint_as_float(w[e / 4][e % 4]);
            }
        }
    }
};
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    store4<T>(p, f32x4{x[0], x[1], x[2], x[3]}, 1.0f);
    store4<T>(p + 4, f32x4{x[4], x[5], x[6], x[7]}, 1.0f);
}

__device__ __forceinline__ int mx_token(int U) {
    const int lane = threadIdx.x & 63, each = 64 / U;
    return lane / U < each ? (int)(threadIdx.x >> 6) * each + lane / U : 64;
}

// Position and cache row of a work-group's tokens t0 .. t1 - 1, by which sequence
// each is of: a sequence that has tokens among them writes its index beside those
// (every thread takes part).
struct MxPlace {
    int pos;                 // negative: left out
    unsigned block, inside;  // of the token; block ~0: past the table or outside the pool
};
__device__ __forceinline__ MxPlace mx_place(const BatchParams &p, int t0, int t1, int k) {
    __shared__ int seq_of[64];  // 256 threads, at least 4 to a token
    const int tid = threadIdx.x;
    if (tid < 64) seq_of[tid] = -1;
    __syncthreads();
    for (int s = tid; s < p.n_seq; s += 256) {
        const int lo = max(p.cu_q[s], t0), hi = min(p.cu_q[s + 1], t1);
        for (int i = lo; i < hi; ++i) seq_of[i - t0] = s;
    }
    __syncthreads();
    MxPlace x{-1, ~0u, 0};
    if (t0 + k >= t1 || k >= 64 || seq_of[k] < 0) return x;
    const int s = seq_of[k];
    const long long at = (long long)p.lens[s] - p.cu_q[s + 1] + t0 + k;  // (may pass 32 bits either way)
    if (at < 0 || at > INT_MAX) return x;
    x.pos = (int)at;
    const int blk = x.pos >> p.bs_shift;
    if (blk >= p.max_blocks) return x;
    const unsigned e = (unsigned)p.table[(long long)s * p.table_stride + blk];
    if (e < (unsigned)p.n_blocks) x.block = e;
    x.inside = (unsigned)x.pos & ((1u << p.bs_shift) - 1u);
    return x;
}

// The largest of the 4 lanes that share 32 elements.
__device__ __forceinline__ unsigned mx_quad_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));
}

// Chunk u (8 elements) of a head's row into the cache: codes, and E from the first
// of each 4 lanes.
template <int BITS>
__device__ __forceinline__ void mx_put(char *codes, char *scales, int u, float (&x)[8]) {
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    most = mx_quad_max(most);
    // largest 1.f 2^n: E = n + 127 - 2 (4 bits) or - 8, one more where 1.f is above 1.75
    int E = max((int)((most + 0x1fffffu) >> 23) - (BITS == 4 ? 2 : 8), kMxLeast);
    // (for the wave: a branch of single lanes would copy x)
    if (__builtin_amdgcn_ballot_w64(most > 0x7f600000u) != 0) {  // 1.75 2^127: what is above would round to 2^128
        if (most > 0x7f600000u) E = BITS == 4 ? 252 : 246;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = __builtin_fminf(__builtin_fmaxf(x[e], -0x1.cp127f), 0x1.cp127f);
            x[e] = most >= 0x7f800000u ? 0.f : y;
        }
    }
    const float power = mx_power(E);
    if (most >= 0x7f800000u) E = 255;
    if constexpr (BITS == 4) {  // (6 2^(E - 127) and more saturate)
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], power, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], power, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], power, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], power, 3);
        *reinterpret_cast<uint32_t *>(codes + 4 * u) = w;
    } else {
        i16x2 a{0, 0}, b{0, 0};
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, x[0], x[1], power, false);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, x[2], x[3], power, true);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, x[4], x[5], power, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, x[6], x[7], power, true);
        *reinterpret_cast<u32x2 *>(codes + 8 * u) =
            u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
    if ((u & 3) == 0) scales[u >> 2] = (char)E;
}

// Which rows and heads a thread of the append has: tokens of a work-group, U threads
// each, and a group of heads of Q, of K (the grid's y past Q's groups) or of V
// (past K's): each then is a loop without branches between them, and Q needs no 64
// bits.
struct MxWalk {
    int t0, t1, k, u;         // tokens, the thread's among them, its number there
    int of, first, last;      // Q, K or V, its heads
    bool mine;
    __device__ __forceinline__ MxWalk(const BatchParams &p, int U) {
        t0 = (int)blockIdx.x * mx_tokens(U);
        t1 = min(t0 + mx_tokens(U), p.n_tok);
        k = mx_token(U);
        u = (threadIdx.x & 63) % U;
        mine = k < 64 && t0 + k < t1;
        const int qg = (p.Hq + p.hpt - 1) / p.hpt, kg = (p.Hkv + p.hpt_kv - 1) / p.hpt_kv, y = blockIdx.y;
        of = y < qg ? 0 : y < qg + kg ? 1 : 2;
        first = of == 0 ? y * p.hpt : (y - qg - (of - 1) * kg) * p.hpt_kv;
        last = of == 0 ? min(first + p.hpt, p.Hq) : min(first + p.hpt_kv, p.Hkv);
    }
    template <class T>
    __device__ __forceinline__ const T *in(const BatchParams &p) const {
        return static_cast<const T *>(p.q) + (long long)(t0 + k) * p.q_rs + (of == 0 ? 0 : p.Hq + (of - 1) * p.Hkv) * p.d;
    }
    // load(j, head) for up to AHEAD heads together (the first of them before
    // search(), which says whether there is a place), then put(j, head)
    template <int AHEAD, class Load, class Search, class Put>
    __device__ __forceinline__ void run(Load load, Search search, Put put) const {
        auto each = [&](int h, auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (h + j < last) f(j, h + j);
            }
        };
        if (mine) each(first, load);
        if (!search()) return;
        for (int h = first; h < last; h += AHEAD) {
            if (h > first) each(h, load);
            each(h, put);
        }
    }
};

// Where the codes and E of a token's rows of KV head `head` begin.
struct MxRow {
    char *codes, *scales;
};
template <int BITS>
__device__ __forceinline__ MxRow mx_row_of(const BatchParams &p, const MxPlace &at, void *pool, int head) {
    const MxHead m = mx_head(p, head);
    char *block = static_cast<char *>(pool) + (size_t)at.block * (unsigned)p.kv_rs;
    return MxRow{block + m.codes + at.inside * mx_code_bytes(p.d, BITS), block + m.scales + at.inside * mx_scale_bytes(p.d)};
}

// Whole rows turned in halves (dim = d, a multiple of 64): a thread has 8 elements of
// the first half and their partners of the second. us: 5400 tokens of 32/8 heads, d =
// 128, 4 bits, 116 MB: 29 (4.0 TB/s; the ordinary append, 132 MB, 32); 16 tokens of
// 14/2 heads 4.7 (4.0). With 8 elements to a thread, as below, where each angle is
// formed twice: 35 and 5.4. Large calls are bound by memory, small ones by the chain
// of loads (cu_q, length, block) and the angles in 64 bits behind it.
template <class T, int BITS>
__device__ __forceinline__ void append_halves(const BatchParams &p, double factor) {
    constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1;  // (4 and 2: the same time)
    const int half = p.d / 2;
    const MxWalk w(p, p.d / 16);
    const T *in = w.in<T>(p) + 8 * w.u;
    double freq[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) freq[e] = w.of < 2 ? p.freq[8 * w.u + e] : 0.0;
    Raw8<T> xr[AHEAD], yr[AHEAD];
    MxPlace at;
    auto load = [&](int j, int h) __attribute__((always_inline)) {
        xr[j].load(in + h * p.d);
        yr[j].load(in + h * p.d + half);
    };
    auto search = [&]() __attribute__((always_inline)) {
        at = mx_place(p, w.t0, w.t1, w.k);
        return at.pos >= 0 && (w.of == 0 || at.block != ~0u);
    };
    auto quantise = [&](void *pool, int h, float (&x)[8], float (&y)[8]) __attribute__((always_inline)) {
        const MxRow r = mx_row_of<BITS>(p, at, pool, h);
        mx_put<BITS>(r.codes, r.scales, w.u, x);
        mx_put<BITS>(r.codes, r.scales, w.u + half / 8, y);
    };
    if (w.of == 0) {
        float c[8], s[8];
        T *out = static_cast<T *>(p.o) + (long long)(w.t0 + w.k) * p.o_rs + 8 * w.u;
        w.run<AHEAD>(
            load,
            [&]() __attribute__((always_inline)) {
                if (!search()) return false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    turn_angle((double)at.pos * (freq[e] * kTurn), c[e], s[e]);
                    c[e] *= (float)factor;
                    s[e] *= (float)factor;
                }
                return true;
            },
            [&](int j, int h) __attribute__((always_inline)) {
                float x[8], y[8], a[8], b[8];
                xr[j].get(x);
                yr[j].get(y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] = x[e] * c[e] - y[e] * s[e];
                    b[e] = y[e] * c[e] + x[e] * s[e];
                }
                store8<T>(out + h * p.d, a);
                store8<T>(out + h * p.d + half, b);
            });
    } else if (w.of == 1) {
        double c[8], s[8];
        w.run<AHEAD>(
            load,
            [&]() __attribute__((always_inline)) {
                if (!search()) return false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    turn_angle64((double)at.pos * (freq[e] * kTurn), c[e], s[e]);
                    c[e] *= factor;
                    s[e] *= factor;
                }
                return true;
            },
            [&](int j, int h) __attribute__((always_inline)) {
                float x[8], y[8];
                xr[j].get(x);
                yr[j].get(y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double u = x[e], v = y[e];
                    x[e] = (float)__builtin_fma(u, c[e], -v * s[e]);
                    y[e] = (float)__builtin_fma(v, c[e], u * s[e]);
                }
                quantise(p.k, h, x, y);
            });
    } else {
        w.run<AHEAD>(load, search, [&](int j, int h) __attribute__((always_inline)) {
            float x[8], y[8];
            xr[j].get(x);
            yr[j].get(y);
            quantise(p.v, h, x, y);
        });
    }
}

// Any other rotation (interleaved, of a part of the row, of odd sizes, or none): a
// thread has 8 elements, element e0 + e turns with element `with`: y = x c + with s.
template <class T, int BITS>
__device__ __forceinline__ void append_any(const BatchParams &p, double factor) {
    const MxWalk w(p, p.d / 8);
    const T *in = w.in<T>(p);
    const int e0 = 8 * w.u, half = p.dim / 2;
    const bool turned = w.of < 2 && p.dim > 0;
    Raw8<T> xr;
    MxPlace at;
    double c[8], s[8];
    T *out = static_cast<T *>(p.o) + (long long)(w.t0 + w.k) * p.o_rs + e0;
    w.run<1>(
        [&](int, int h) __attribute__((always_inline)) { xr.load(in + h * p.d + e0); },
        [&]() __attribute__((always_inline)) {
            at = mx_place(p, w.t0, w.t1, w.k);
            if (at.pos < 0 || (w.of > 0 && at.block == ~0u)) return false;
            if (turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = e0 + e;
                    const bool second = p.interleaved ? i & 1 : i >= half;
                    const int pair = i >= p.dim ? 0 : p.interleaved ? i >> 1 : second ? i - half : i;
                    turn_angle64((double)at.pos * (p.freq[pair] * kTurn), c[e], s[e]);
                    c[e] *= factor;
                    s[e] = (second ? s[e] : -s[e]) * factor;
                }
            }
            return true;
        },
        [&](int, int h) __attribute__((always_inline)) {
            float x[8], y[8];
            xr.get(x);
            if (turned) {
                const T *row = in + h * p.d;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = e0 + e, with = i >= p.dim ? i : p.interleaved ? i ^ 1 : i < half ? i + half : i - half;
                    if constexpr (sizeof(T) == 2) y[e] = __uint_as_float((uint32_t)row[with] << 16);
                    else y[e] = row[with];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float r = (float)__builtin_fma((double)x[e], c[e], (double)y[e] * s[e]);
                    x[e] = e0 + e < p.dim ? r : x[e];
                }
            }
            if (w.of == 0) {
                // (q_out may be qkv: the wave has all of the row's partners before it stores)
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                store8<T>(out + h * p.d, x);
            } else {
                const MxRow r = mx_row_of<BITS>(p, at, w.of == 1 ? p.k : p.v, h);
                mx_put<BITS>(r.codes, r.scales, w.u, x);
            }
        });
}

// Row r of k_out and v_out is what the cache holds at the r-th row's position (as the
// append counts them): a thread has 8 elements of a token's rows and walks heads,
// the loads of 8 together. The rows are not read again here: stored past the caches.
// Bound by memory: 12 sequences of 2000-16384, 8 heads of 128, 4 bits to bf16 (0.69
// GB): 128 us, 5.4 TB/s (a copy 5.1); 136 with ordinary stores, 148 head by head.
template <class T, int BITS>
__device__ __forceinline__ void read_mx_body(const BatchParams &p, void *v_out) {
    const int U = p.d / 8, per = mx_tokens(U);
    const int t0 = (int)blockIdx.x * per, t1 = min(t0 + per, p.n_tok);
    const int u = (threadIdx.x & 63) % U, k = mx_token(U);
    const MxPlace at = mx_place(p, t0, t1, k);
    if (at.block == ~0u) return;
    const int h0 = (int)blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, 2 * p.Hkv);
    const size_t block = (size_t)at.block * (unsigned)p.kv_rs;
    constexpr int AHEAD = 8;
    for (int h = h0; h < h1; h += AHEAD) {
        uint32_t w[AHEAD][BITS / 4];
        unsigned E[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (h + j >= h1) break;
            const bool of_k = h + j < p.Hkv;
            const MxHead m = mx_head(p, of_k ? h + j : h + j - p.Hkv);
            const char *x = static_cast<const char *>(of_k ? p.k : p.v) + block;
            load_words(w[j], x + m.codes + at.inside * mx_code_bytes(p.d, BITS) + BITS * u);
            E[j] = (unsigned char)x[m.scales + at.inside * mx_scale_bytes(p.d) + (u >> 2)];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (h + j >= h1) break;
            const bool of_k = h + j < p.Hkv;
            const bf16x8 v = mx_values<BITS>(w[j], mx_power(E[j]));
            T *out = static_cast<T *>(of_k ? p.o : v_out) + (long long)(t0 + k) * p.o_rs + (of_k ? h + j : h + j - p.Hkv) * p.d + 8 * u;
            if constexpr (sizeof(T) == 2) {
                __builtin_nontemporal_store(v, reinterpret_cast<bf16x8 *>(out));
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    __builtin_nontemporal_store(f32x4{(float)v[i], (float)v[i + 1], (float)v[i + 2], (float)v[i + 3]},
                                                reinterpret_cast<f32x4 *>(out + i));
            }
        }
    }
}

#define MXFA_MX(BITS, SUFFIX, T)                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void mxfa_append_x##BITS##SUFFIX(BatchParams p, double factor) {      \
        append_halves<T, BITS>(p, factor);                                                                      \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void mxfa_append_x##BITS##SUFFIX##1(BatchParams p, double factor) {   \
        append_any<T, BITS>(p, factor);                                                                     \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void mxfa_read_x##BITS##SUFFIX(BatchParams p, void *v_out) {          \
        read_mx_body<T, BITS>(p, v_out);                                                                               \
    }
MXFA_MX(8, b, u16)
MXFA_MX(8, f, float)
MXFA_MX(4, b, u16)
MXFA_MX(4, f, float)
#undef MXFA_MX
#endif

// Heads per thread: as many as leave `threads`, so that a thread's angles and place
// serve many heads of a large call and a small one still spreads over the GPU. us, 5400
// tokens of 32/8 heads, d = 128: append 29 by 2^17, 33 by 2^18; read 7.1 by 2^18, 8.1 by
// 2^17.
static int mx_heads_per_thread(long long units, int heads, long long threads) {
    return (int)std::clamp<long long>(units * heads / threads, 1, heads);
}

hipError_t launch_append_mx(BatchParams p, double factor, int dtype_bf16, hipStream_t stream) {
    static constexpr KernelId ids[2][2][2] = {{{k_mxfa_append_x8f, k_mxfa_append_x8f1}, {k_mxfa_append_x8b, k_mxfa_append_x8b1}},
                                              {{k_mxfa_append_x4f, k_mxfa_append_x4f1}, {k_mxfa_append_x4b, k_mxfa_append_x4b1}}};
    const bool halves = !p.interleaved && p.dim == p.d && p.d % 64 == 0;
    const int U = p.d / (halves ? 16 : 8), per = mx_tokens(U);
    p.hpt = std::min(mx_heads_per_thread((long long)p.n_tok * U, p.Hq + 2 * p.Hkv, 1 << 17), p.Hq);
    p.hpt_kv = std::min(p.hpt, p.Hkv);
    const int groups = (p.Hq + p.hpt - 1) / p.hpt + 2 * ((p.Hkv + p.hpt_kv - 1) / p.hpt_kv);
    void *args[] = {&p, &factor};
    return launch_kernel(ids[p.bits == 4][dtype_bf16 != 0][!halves], dim3((p.n_tok + per - 1) / per, groups), dim3(256), args,
                         stream);
}

hipError_t launch_read_mx(BatchParams p, void *v_out, int dtype_bf16, hipStream_t stream) {
    static constexpr KernelId ids[2][2] = {{k_mxfa_read_x8f, k_mxfa_read_x8b}, {k_mxfa_read_x4f, k_mxfa_read_x4b}};
    const int U = p.d / 8, per = mx_tokens(U), H = 2 * p.Hkv;
    p.hpt = mx_heads_per_thread((long long)p.n_tok * U, H, 1 << 18);
    void *args[] = {&p, &v_out};
    return launch_kernel(ids[p.bits == 4][dtype_bf16 != 0], dim3((p.n_tok + per - 1) / per, (H + p.hpt - 1) / p.hpt),
                         dim3(256), args, stream);
}

}  // namespace mxfa
