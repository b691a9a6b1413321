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

// 8 neighbouring elements.
template <class T>
__device__ __forceinline__ void load8(float (&x)[8], const T *p) {
    if constexpr (sizeof(T) == 2) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    }
}
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
    if (most > 0x7f600000u) {  // 1.75 2^127: what is above would round to 2^128
        E = BITS == 4 ? 252 : 246;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = most >= 0x7f800000u ? 0.f : __builtin_fminf(__builtin_fmaxf(x[e], -0x1.cp127f), 0x1.cp127f);
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

// A thread has 8 elements of a token's rows and walks heads h0 .. h1 - 1 of [Q heads
// | K heads | V heads] with their angles. WHOLE: the rotated part and its halves are
// whole chunks, so what an element turns with is a chunk too.
template <class T, int BITS, bool WHOLE>
__device__ __forceinline__ void append_mx_body(const BatchParams &p, double factor) {
    const int U = p.d / 8, per = mx_tokens(U);
    const int t0 = (int)blockIdx.x * per, t1 = min(t0 + per, p.n_tok);
    const int u = (threadIdx.x & 63) % U, e0 = 8 * u, k = mx_token(U);
    const MxPlace at = mx_place(p, t0, t1, k);
    if (at.pos < 0) return;
    const int h0 = (int)blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.Hq + 2 * p.Hkv);
    const T *in = static_cast<const T *>(p.q) + (long long)(t0 + k) * p.q_rs;
    // element e0 + e turns with element `with[e]`: y = x c + with s
    const int half = p.dim / 2;
    double c[8], s[8];
    int with[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at_e = e0 + e;
        c[e] = 1.0;
        s[e] = 0.0;
        with[e] = at_e;
        if (at_e >= p.dim) continue;
        const bool second = p.interleaved ? at_e & 1 : at_e >= half;
        const int pair = p.interleaved ? at_e >> 1 : second ? at_e - half : at_e;
        with[e] = p.interleaved ? at_e ^ 1 : second ? at_e - half : at_e + half;
        double cs, sn;
        turn_angle64((double)at.pos * (p.freq[pair] * 0.15915494309189535), cs, sn);
        c[e] = cs * factor;
        s[e] = (second ? sn : -sn) * factor;
    }
    for (int h = h0; h < h1; ++h) {
        const int kv = h - p.Hq;
        if (kv >= 0 && at.block == ~0u) break;
        const T *row = in + h * p.d;
        float x[8], y[8];
        load8<T>(x, row + e0);
        const bool turns = kv < p.Hkv && e0 < p.dim;
        if (turns) {
            if (WHOLE && p.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
            } else if (WHOLE) {
                load8<T>(y, row + with[0]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (sizeof(T) == 2) y[e] = __uint_as_float((uint32_t)row[with[e]] << 16);
                    else y[e] = row[with[e]];
                }
            }
        }
        if (kv < 0) {
            if (turns) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = WHOLE || e0 + e < p.dim ? x[e] * (float)c[e] + y[e] * (float)s[e] : x[e];
            }
            store8<T>(static_cast<T *>(p.o) + (long long)(t0 + k) * p.o_rs + h * p.d + e0, x);
            continue;
        }
        if (turns) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = WHOLE || e0 + e < p.dim ? (float)__builtin_fma((double)x[e], c[e], (double)y[e] * s[e]) : x[e];
        }
        const MxHead m = mx_head(p, kv < p.Hkv ? kv : kv - p.Hkv);
        char *block = static_cast<char *>(kv < p.Hkv ? p.k : p.v) + (size_t)at.block * (unsigned)p.kv_rs;
        mx_put<BITS>(block + m.codes + at.inside * mx_code_bytes(p.d, BITS), block + m.scales + at.inside * mx_scale_bytes(p.d),
                     u, x);
    }
}

// Row r of k_out and v_out is what the cache holds at the r-th row's position (as the
// append counts them): a thread has 8 elements of a token's rows and walks heads.
template <class T, int BITS>
__device__ __forceinline__ void read_mx_body(const BatchParams &p, void *v_out) {
    const int U = p.d / 8, per = mx_tokens(U);
    const int t0 = (int)blockIdx.x * per, t1 = min(t0 + per, p.n_tok);
    const int u = (threadIdx.x & 63) % U, k = mx_token(U);
    const MxPlace at = mx_place(p, t0, t1, k);
    if (at.block == ~0u) return;
    const int h0 = (int)blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, 2 * p.Hkv);
    for (int h = h0; h < h1; ++h) {
        const int head = h < p.Hkv ? h : h - p.Hkv;
        const MxHead m = mx_head(p, head);
        const char *block = static_cast<const char *>(h < p.Hkv ? p.k : p.v) + (size_t)at.block * (unsigned)p.kv_rs;
        uint32_t w[BITS / 4];
        load_words(w, block + m.codes + at.inside * mx_code_bytes(p.d, BITS) + BITS * u);
        const unsigned E = (unsigned char)block[m.scales + at.inside * mx_scale_bytes(p.d) + (u >> 2)];
        const bf16x8 v = mx_values<BITS>(w, mx_power(E));
        T *out = static_cast<T *>(h < p.Hkv ? p.o : v_out) + (long long)(t0 + k) * p.o_rs + head * p.d + 8 * u;
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<bf16x8 *>(out) = v;
        } else {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
            store8<T>(out, x);
        }
    }
}

#define MXFA_MX(BITS, SUFFIX, T)                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void mxfa_append_x##BITS##SUFFIX(BatchParams p, double factor) {      \
        append_mx_body<T, BITS, true>(p, factor);                                                                      \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void mxfa_append_x##BITS##SUFFIX##1(BatchParams p, double factor) {   \
        append_mx_body<T, BITS, false>(p, factor);                                                                     \
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

// Heads per thread: as many as leave 2^18 threads (the ordinary append's rule).
static int mx_heads_per_thread(long long units, int heads) {
    return (int)std::clamp<long long>(units * heads / (1 << 18), 1, heads);
}

hipError_t launch_append_mx(BatchParams p, double factor, int dtype_bf16, hipStream_t stream) {
    static constexpr KernelId ids[2][2][2] = {{{k_mxfa_append_x8f, k_mxfa_append_x8f1}, {k_mxfa_append_x8b, k_mxfa_append_x8b1}},
                                              {{k_mxfa_append_x4f, k_mxfa_append_x4f1}, {k_mxfa_append_x4b, k_mxfa_append_x4b1}}};
    const int U = p.d / 8, per = mx_tokens(U), H = p.Hq + 2 * p.Hkv;
    p.hpt = mx_heads_per_thread((long long)p.n_tok * U, H);
    const bool whole = p.dim % (p.interleaved ? 8 : 16) == 0;
    void *args[] = {&p, &factor};
    return launch_kernel(ids[p.bits == 4][dtype_bf16 != 0][!whole], dim3((p.n_tok + per - 1) / per, (H + p.hpt - 1) / p.hpt),
                         dim3(256), args, stream);
}

hipError_t launch_read_mx(BatchParams p, void *v_out, int dtype_bf16, hipStream_t stream) {
    static constexpr KernelId ids[2][2] = {{k_mxfa_read_x8f, k_mxfa_read_x8b}, {k_mxfa_read_x4f, k_mxfa_read_x4b}};
    const int U = p.d / 8, per = mx_tokens(U), H = 2 * p.Hkv;
    p.hpt = mx_heads_per_thread((long long)p.n_tok * U, H);
    void *args[] = {&p, &v_out};
    return launch_kernel(ids[p.bits == 4][dtype_bf16 != 0], dim3((p.n_tok + per - 1) / per, (H + p.hpt - 1) / p.hpt),
                         dim3(256), args, stream);
}

}  // namespace mxfa
