// Rotary positions, and the write of new tokens into a paged KV cache.
//
// Pair i of a head's first `dim` elements, (x1, x2) = (x[i], x[i + dim / 2])
// or, interleaved, (x[2i], x[2i + 1]), turns by the angle a = position freq[i]:
//     y1 = f (x1 cos a - x2 sin a),   y2 = f (x2 cos a + x1 sin a);
// elements dim .. d - 1 are copied. The gradient is the transpose, the same
// with -a. Products and sums are in fp32 and rounded once.
//
// Bound: memory, each head read and written once (2 flops a byte at most). A
// thread has one unit of a row, two 16-byte chunks of pairs or one of the
// copied rest, computes its angles once and walks hpt heads with them: no table
// of cosines is read or kept, and the angles' 64-bit arithmetic hides behind the
// first loads (B4, 12 + 12 heads, N4096, d = 64 bf16, 100 MB: 18 us, a copy 20; fp32, 200
// MB: 44, 4.6 TB/s). A short call stays below the copy's rate: fp32, B3, 10 + 10
// heads, N777, 24 MB: 6.6 us (3.6 TB/s), and 7.2 where half of each row is only
// copied: of a row's 12 threads then 4 have pairs and angles and 8 a single chunk.
#include <limits.h>

#include <algorithm>

#include "fa_cache.h"
#include "fa_launch.h"

namespace mxfa {

// cos and sin of a whole angle given in turns, off by about 1.2e-7 at most, and by
// what the angle itself is: the position times the frequency is formed, rounded
// three times (with 1 / 2 pi), in 64 bits, so by up to 3 x 2^-53 of the angle (a
// position of 2^20 at a frequency of 1 3.5e-10 radians, of 2^31 7e-7; in 32 bits
// 2^20 would be off by 0.06). It is reduced to [-1/8, 1/8] turns there, then
// Taylor's series, whose first terms left out are z^11 / 11! <= 1.8e-9 and
// z^12 / 12! <= 1.2e-10 at z = pi / 4.
__device__ __forceinline__ void turn_angle(double turns, float &c, float &s) {
    turns -= __builtin_rint(turns);
    const double quarter = __builtin_rint(4.0 * turns);
    const float z = 6.283185307179586f * (float)__builtin_fma(-0.25, quarter, turns);
    const int q = (int)quarter & 3;  // (quarter: -2 .. 2)
    const float w = z * z;
    float sn = __builtin_fmaf(w, 2.75573192e-6f, -1.98412698e-4f);
    sn = __builtin_fmaf(w, sn, 8.33333333e-3f);
    sn = __builtin_fmaf(w, sn, -1.66666667e-1f);
    sn = __builtin_fmaf(z * w, sn, z);
    float cs = __builtin_fmaf(w, -2.75573192e-7f, 2.48015873e-5f);
    cs = __builtin_fmaf(w, cs, -1.38888889e-3f);
    cs = __builtin_fmaf(w, cs, 4.16666667e-2f);
    cs = __builtin_fmaf(w, cs, -0.5f);
    cs = __builtin_fmaf(w, cs, 1.0f);
    const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
    c = q == 1 || q == 2 ? -a : a;
    s = q >= 2 ? -b : b;
}

constexpr double kTurn = 0.15915494309189535;  // 1 / (2 pi)

// VEC elements of type T as floats: 16 bytes, or 8 or a single element where
// the rotated part is no whole number of those.
template <class T, int VEC>
struct Chunk;
template <>
struct Chunk<u16, 8> {
    uint4 r;
    __device__ __forceinline__ void load(const u16 *p) { r = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(u16 *p) const { *reinterpret_cast<uint4 *>(p) = r; }
    __device__ __forceinline__ float get(int e) const {
        const uint32_t w = (&r.x)[e >> 1];
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void set(int e, float a, float b) {  // elements e, e + 1 (e even)
        (&r.x)[e >> 1] = (uint32_t)to_bf16_bits(a) | ((uint32_t)to_bf16_bits(b) << 16);
    }
};
template <>
struct Chunk<u16, 4> {
    uint2 r;
    __device__ __forceinline__ void load(const u16 *p) { r = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void store(u16 *p) const { *reinterpret_cast<uint2 *>(p) = r; }
    __device__ __forceinline__ float get(int e) const {
        const uint32_t w = e < 2 ? r.x : r.y;
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void set(int e, float a, float b) {
        (e < 2 ? r.x : r.y) = (uint32_t)to_bf16_bits(a) | ((uint32_t)to_bf16_bits(b) << 16);
    }
};
template <>
struct Chunk<float, 4> {
    float4 r;
    __device__ __forceinline__ void load(const float *p) { r = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = r; }
    __device__ __forceinline__ float get(int e) const { return (&r.x)[e]; }
    __device__ __forceinline__ void set(int e, float a, float b) {
        (&r.x)[e] = a;
        (&r.x)[e + 1] = b;
    }
};
template <class T>
struct Chunk<T, 1> {
    T r;
    __device__ __forceinline__ void load(const T *p) { r = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = r; }
    __device__ __forceinline__ float get(int) const {
        if constexpr (sizeof(T) == 2) return __uint_as_float((uint32_t)r << 16);
        else return r;
    }
    __device__ __forceinline__ void put(float a) {
        if constexpr (sizeof(T) == 2) r = to_bf16_bits(a);
        else r = a;
    }
};

// The two chunks of one unit of pairs, turned in place.
template <class T, int VEC>
__device__ __forceinline__ void turn(Chunk<T, VEC> &a, Chunk<T, VEC> &b, const float (&c)[VEC], const float (&s)[VEC],
                                     int interleaved) {
    if constexpr (VEC == 1) {
        const float x = a.get(0), y = b.get(0);
        a.put(x * c[0] - y * s[0]);
        b.put(y * c[0] + x * s[0]);
    } else {
        if (interleaved) {
            // chunk a holds pairs 0 .. VEC / 2 - 1 of the unit, b the rest
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const int i = e / 2, j = VEC / 2 + e / 2;
                const float x = a.get(e), y = a.get(e + 1), u = b.get(e), v = b.get(e + 1);
                a.set(e, x * c[i] - y * s[i], y * c[i] + x * s[i]);
                b.set(e, u * c[j] - v * s[j], v * c[j] + u * s[j]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float x0 = a.get(e), x1 = a.get(e + 1), y0 = b.get(e), y1 = b.get(e + 1);
                a.set(e, x0 * c[e] - y0 * s[e], x1 * c[e + 1] - y1 * s[e + 1]);
                b.set(e, y0 * c[e] + x0 * s[e], y1 * c[e + 1] + x1 * s[e + 1]);
            }
        }
    }
}

// The units of a row: dim / (2 VEC) of pairs, then the rest in single chunks.
template <int VEC>
__host__ __device__ constexpr int rotary_units(int d, int dim) {
    return dim / (2 * VEC) + (d - dim) / VEC;
}

// Unit u of a row: where its chunks lie, and, once `at` was called, its angles at a
// position.
template <class T, int VEC>
struct Unit {
    int e0, e1;  // first elements of the chunks (e1 < 0: a single chunk, copied)
    float c[VEC], s[VEC];
    __device__ __forceinline__ Unit(int u, int dim, int interleaved) {
        const int nr = dim / (2 * VEC);
        e0 = u >= nr ? dim + (u - nr) * VEC : interleaved ? 2 * VEC * u : VEC * u;
        e1 = u >= nr ? -1 : interleaved ? e0 + VEC : e0 + dim / 2;
    }
    __device__ __forceinline__ void at(int u, const double *freq, int pos, float factor, float sin_sign) {
        if (e1 < 0) return;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            turn_angle((double)pos * (freq[VEC * u + e] * kTurn), c[e], s[e]);
            c[e] *= factor;
            s[e] *= factor * sin_sign;
        }
    }
};

// A thread's heads h0 .. h1 - 1 of a row, the chunks at e0 and (e1 >= 0) e1 of each:
// from(h) is where head h is read, put(h, x, y) turns and stores it. The loads of
// kHeadsAhead heads go out together, and the first of them before first(), which
// finds what put needs.
constexpr int kHeadsAhead = 4;
template <class T, int VEC, class From, class First, class Put>
__device__ __forceinline__ void walk_heads(int h0, int h1, int e0, int e1, From from, First first, Put put) {
    Chunk<T, VEC> x[kHeadsAhead], y[kHeadsAhead];
    auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kHeadsAhead; ++j) {
            if (h + j >= h1) break;
            const T *row = from(h + j);
            x[j].load(row + e0);
            if (e1 >= 0) y[j].load(row + e1);
        }
    };
    load(h0);
    first();
    for (int h = h0; h < h1; h += kHeadsAhead) {
        if (h > h0) load(h);
#pragma unroll
        for (int j = 0; j < kHeadsAhead; ++j) {
            if (h + j >= h1) break;
            put(h + j, x[j], y[j]);
        }
    }
}

// Grid: (units of all tokens in work-groups of 256, heads of Q then K in
// groups of hpt, batches).
template <class T, int VEC>
__device__ __forceinline__ void rotary_body(const RotaryParams &p) {
    const int U = rotary_units<VEC>(p.d, p.dim);
    const unsigned i = blockIdx.x * 256 + threadIdx.x;  // N U stays below 2^31
    const int n = (int)(i / (unsigned)U), u = (int)(i - (unsigned)n * (unsigned)U);
    if (n >= p.N) return;
    const int b = blockIdx.z;
    Unit<T, VEC> un(u, p.dim, p.interleaved);
    const int h0 = (int)blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.H[0] + p.H[1]);
    walk_heads<T, VEC>(
        h0, h1, un.e0, un.e1,
        [&](int h) __attribute__((always_inline)) {
            const int t = h >= p.H[0], hh = h - (t ? p.H[0] : 0);
            const HeadView &v = p.x[t];
            return static_cast<const T *>(v.in) + b * v.in_bs + hh * v.in_hs + n * v.in_ts;
        },
        [&]() __attribute__((always_inline)) {
            un.at(u, p.freq, p.positions != nullptr ? p.positions[b * p.pos_bs + n] : p.pos0 + n, p.factor, p.sin_sign);
        },
        [&](int h, Chunk<T, VEC> &x, Chunk<T, VEC> &y) __attribute__((always_inline)) {
            const int t = h >= p.H[0], hh = h - (t ? p.H[0] : 0);
            const HeadView &v = p.x[t];
            T *row = static_cast<T *>(v.out) + b * v.out_bs + hh * v.out_hs + n * v.out_ts;
            if (un.e1 >= 0) {
                turn<T, VEC>(x, y, un.c, un.s, p.interleaved);
                y.store(row + un.e1);
            }
            x.store(row + un.e0);
        });
}

// The cache append: rows of [Q heads | K heads | V heads] of new tokens; Q is
// turned into p.o, K is turned and V copied into the cache rows of the tokens'
// positions. A work-group has 256 / U tokens (the grid's y: head groups of hpt);
// it first finds each token's sequence: every sequence that has tokens among
// them writes its index beside those, so the search costs one load of cu_q
// instead of a bisection's chain of them. Bound by memory where there are many
// tokens (5400 of 32/8 heads, d = 128, 132 MB: 23.5 us, 32 from memory that no cache
// holds, where a copy takes 26), by the chain of loads cu_q, length,
// block, row where there are few (16 of 14/2 heads: 4.0 us). fp32, d = 64: 22.4
// (132 MB) and 3.7.
template <class T, int VEC>
__device__ __forceinline__ void append_body(const BatchParams &p) {
    const int U = rotary_units<VEC>(p.d, p.dim), tid = threadIdx.x;  // (U is at most 255)
    const int per = 256 / U;
    __shared__ int seq_of[256];
    const int t0 = (int)blockIdx.x * per, t1 = min(t0 + per, p.n_tok);
    const int k = tid / U, u = tid - k * U, t = t0 + k;
    const bool mine = k < per && t < t1;  // (every thread takes part in the search)
    const int h0 = (int)blockIdx.y * p.hpt, h1 = mine ? min(h0 + p.hpt, p.Hq + 2 * p.Hkv) : h0;
    const T *in = static_cast<const T *>(p.q) + (long long)t * p.q_rs;
    Unit<T, VEC> un(u, p.dim, p.interleaved);
    int pos = -1;
    long long crow = -1;
    auto search = [&]() __attribute__((always_inline)) {
        if (tid < per) seq_of[tid] = -1;
        __syncthreads();
        for (int s = tid; s < p.n_seq; s += 256) {
            const int lo = max(p.cu_q[s], t0), hi = min(p.cu_q[s + 1], t1);
            for (int i = lo; i < hi; ++i) seq_of[i - t0] = s;
        }
        __syncthreads();
        if (!mine || seq_of[k] < 0) return;
        const int s = seq_of[k];
        const long long at = (long long)p.lens[s] - p.cu_q[s + 1] + t;  // (may pass 32 bits either way)
        if (at < 0 || at > INT_MAX) return;
        pos = (int)at;
        const int blk = pos >> p.bs_shift;
        if (blk < p.max_blocks) {
            const int e = p.table[(long long)s * p.table_stride + blk];
            if ((unsigned)e < (unsigned)p.n_blocks)
                crow = ((long long)e << p.bs_shift) + (pos & ((1 << p.bs_shift) - 1));
        }
        un.at(u, p.freq, pos, p.factor, 1.0f);
    };
    walk_heads<T, VEC>(
        h0, h1, un.e0, un.e1, [&](int h) __attribute__((always_inline)) { return in + h * p.d; }, search,
        [&](int h, Chunk<T, VEC> &x, Chunk<T, VEC> &y) __attribute__((always_inline)) {
            const int kv = h - p.Hq;
            if (pos < 0 || (kv >= 0 && crow < 0)) return;
            T *row = kv < 0 ? static_cast<T *>(p.o) + (long long)t * p.o_rs + h * p.d
                     : kv < p.Hkv ? static_cast<T *>(p.k) + crow * p.kv_rs + kv * p.d
                                  : static_cast<T *>(p.v) + crow * p.kv_rs + (kv - p.Hkv) * p.d;
            if (un.e1 >= 0) {
                if (kv < p.Hkv) turn<T, VEC>(x, y, un.c, un.s, p.interleaved);
                y.store(row + un.e1);
            }
            x.store(row + un.e0);
        });
}

#if defined(__HIP_DEVICE_COMPILE__)
#define MXFA_ROTARY(SUFFIX, T, VEC)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void mxfa_rotary_##SUFFIX(RotaryParams p) { rotary_body<T, VEC>(p); } \
    extern "C" __global__ __launch_bounds__(256) void mxfa_append_##SUFFIX(BatchParams p) { append_body<T, VEC>(p); }
MXFA_ROTARY(b, u16, 8)
MXFA_ROTARY(b4, u16, 4)
MXFA_ROTARY(b1, u16, 1)
MXFA_ROTARY(f, float, 4)
MXFA_ROTARY(f1, float, 1)
#undef MXFA_ROTARY
#endif

// Heads per thread: as many as leave 2^18 threads (4 waves on each SIMD), so that a
// thread's angles serve many heads of a large call and a small one still spreads
// over the GPU. us, 5400 tokens of 32/8 heads, d = 128, from memory that no cache
// holds: 32.5 (2^17: 36, 2^19: 36).
static int heads_per_thread(long long units, int heads) {
    const long long want = units * heads / (1 << 18);
    return (int)std::clamp<long long>(want, 1, heads);
}

// The chunks a rotated part is whole units of, two chunks each: 16 bytes, 8
// (bf16), else single elements.
static int rotary_vec(int dim, int dtype_bf16) {
    if (dim % 16 == 0 && dtype_bf16) return 8;
    return dim % 8 == 0 ? 4 : 1;
}

int rotary_row_units(int d, int dim, int dtype_bf16) {
    const int v = rotary_vec(dim, dtype_bf16);
    return v == 8 ? rotary_units<8>(d, dim) : v == 4 ? rotary_units<4>(d, dim) : rotary_units<1>(d, dim);
}

hipError_t launch_rotary(RotaryParams p, int dtype_bf16, hipStream_t stream) {
    const int v = rotary_vec(p.dim, dtype_bf16), U = rotary_row_units(p.d, p.dim, dtype_bf16), H = p.H[0] + p.H[1];
    p.hpt = heads_per_thread((long long)p.B * p.N * U, H);
    const KernelId id = dtype_bf16 ? (v == 8 ? k_mxfa_rotary_b : v == 4 ? k_mxfa_rotary_b4 : k_mxfa_rotary_b1)
                                   : (v == 4 ? k_mxfa_rotary_f : k_mxfa_rotary_f1);
    void *args[] = {&p};
    const dim3 grid((unsigned)(((long long)p.N * U + 255) / 256), (H + p.hpt - 1) / p.hpt, p.B);
    return launch_kernel(id, grid, dim3(256), args, stream);
}

hipError_t launch_append(BatchParams p, int dtype_bf16, hipStream_t stream) {
    const int v = rotary_vec(p.dim, dtype_bf16), U = rotary_row_units(p.d, p.dim, dtype_bf16);
    const int H = p.Hq + 2 * p.Hkv, per = 256 / U;
    p.hpt = heads_per_thread((long long)p.n_tok * U, H);
    const KernelId id = dtype_bf16 ? (v == 8 ? k_mxfa_append_b : v == 4 ? k_mxfa_append_b4 : k_mxfa_append_b1)
                                   : (v == 4 ? k_mxfa_append_f : k_mxfa_append_f1);
    void *args[] = {&p};
    return launch_kernel(id, dim3((p.n_tok + per - 1) / per, (H + p.hpt - 1) / p.hpt), dim3(256), args, stream);
}

}  // namespace mxfa

// the append into a cache of fewer bits, and its read
#include "fa_mx.hip"
