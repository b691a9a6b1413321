// Microscaled caches: the format, and how its values are made and read.
//
// Of each head's row, 32 neighbouring elements share a power of two 2^(E - 127),
// one byte E; an element is a code of 8 bits (e4m3: a sign, 4 exponent and 3
// mantissa bits, at most 448) or 4 (e2m1: +-0, 0.5, 1, 1.5, 2, 3, 4, 6; two to a
// byte, the even element in the low half) and stands for 2^(E - 127) code. These
// are exact in bf16 (3 or 4 significant bits, and E >= 10 keeps the least, 2^-9
// 2^-117, a normal number), so attention multiplies them as they are: the only
// rounding is the one on the way into the cache. gfx950 converts two codes to bf16,
// times such a power, in one instruction.
//
// E is the least by which the largest of the 32 is at most 448 2^(E - 127), or 7
// 2^(E - 127) in 4 bits: up to 7 rounds to 6, off by no more than between 4 and 6,
// and of normal values the rms error is then 0.112 of their size (0.115 with 6 or 8
// for the 7, 0.101 with a scale of its own to each group, which bf16 would have to
// round again). Elements above 1.75 2^127 count as that: the
// codes nearest to them would stand for 2^128. 32 elements that hold an infinity or
// NaN get E = 255 and read back as NaN.
//
// A pool is blocks of block_size tokens, kv_rs bytes apart; in a block the codes of
// all KV heads, [head][token][CB], then their E, [head][token][SB]: a head's tokens
// lie one after another, so a stage of 64 keys reads whole runs of memory.
#pragma once

#include "fa_cache.h"
#include "fa_device.h"

namespace mxfa {

constexpr int kMxGroup = 32, kMxLeast = 10;

// Bytes of a head's row: codes and E.
__host__ __device__ constexpr int mx_code_bytes(int d, int bits) { return d * bits / 8; }
__host__ __device__ constexpr int mx_scale_bytes(int d) { return d / kMxGroup; }

// Where a head's codes and E begin in a block.
struct MxHead {
    unsigned codes, scales;
};
__host__ __device__ inline MxHead mx_head(const BatchParams &p, int head) {
    const unsigned bs = 1u << p.bs_shift, cb = mx_code_bytes(p.d, p.bits), sb = mx_scale_bytes(p.d);
    return MxHead{(unsigned)head * bs * cb, (unsigned)p.Hkv * bs * cb + (unsigned)head * bs * sb};
}

#if defined(__HIP_DEVICE_COMPILE__)

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 2^(E - 127), infinite for E = 255 (the conversions give NaN then; E = 0, which is
// never written, counts as 2^-127 there)
__device__ __forceinline__ float mx_power(unsigned E) { return __uint_as_float(E << 23); }

// 8 codes, BITS / 4 words from w, as bf16, times `power`.
template <int BITS>
__device__ __forceinline__ bf16x8 mx_values(const uint32_t *w, float power) {
    u32x4 v;
    if constexpr (BITS == 4) {
        v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], power, 0));
        v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], power, 1));
        v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], power, 2));
        v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], power, 3));
    } else {
        v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], power, false));
        v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], power, true));
        v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], power, false));
        v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], power, true));
    }
    return __builtin_bit_cast(bf16x8, v);
}

// N words from p, N a power of two (p aligned to 4 N bytes, 16 at most).
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const void *p) {
    if constexpr (N == 1) {
        w[0] = *static_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const u32x2 x = *static_cast<const u32x2 *>(p);
        w[0] = x[0];
        w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 x = static_cast<const u32x4 *>(p)[i / 4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i + e] = x[e];
        }
    }
}

#endif

}  // namespace mxfa
