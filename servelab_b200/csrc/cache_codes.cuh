// Codes of an 8-bit cache as numbers of 16 bits, exactly, and what goes with products in them.
//
// Both kinds become float16 (11 significant bits against 8 of an 8-bit integer and 4 of e4m3), which costs 5 instructions
// for four int8 codes and 2 for four e4m3 codes (into bfloat16: 7 and 9).  float16's range needs two powers of two:
//   * queries are scaled so that the largest element of a row (in the tcgen05 kernel of a tile of rows, as long as each row's
//     lies within 2^16 of it) lies in [2^13, 2^14): bfloat16 elements down to 2^-28 of it stay exact, what is smaller loses bits
//     that the float32 sums do not have;
//   * a probability 2^(s - m) is taken against a reference m that counts value scales too: m follows the largest
//     s + log2(scale) of the keys that the row sees (lazily: by 2^8).  Then probability x scale x 2^7 is at most 2^15, keys
//     whose contribution is down to 2^-21 of the largest keep all bits of a float16, and the sum of the probabilities,
//     in float32, has the same reference and cancels it.  (A scale of less than 2^-100 counts as 2^-100 there, one of more
//     than 2^110 as that.)  Where scores reach 2^24 a sum with them is off by any power of two: the reference is kept in two
//     numbers there, the largest score and, relative to it, the largest score + log2(scale).
#pragma once

#include <cuda_fp16.h>

#include "cache_attention.cuh"

namespace slb_codes {

// Whether four neighbouring codes come out in the order 0, 2, 1, 3 (otherwise 0, 1, 2, 3).
template <int KIND> __host__ __device__ constexpr bool swaps() { return KIND == CACHE_INT8; }

// Four codes as two pairs of float16.
// int8: 0x6400 | (code ^ 0x80) is 1024 + 128 + code; pairs (0, 2) and (1, 3).   e4m3: pairs (0, 1) and (2, 3).
template <int KIND> __device__ __forceinline__ void four(unsigned x, unsigned& lo, unsigned& hi) {
    if constexpr (KIND == CACHE_INT8) {
        const unsigned a = (x & 0x00FF00FFu) ^ 0x64806480u, b = (x >> 8 & 0x00FF00FFu) ^ 0x64806480u;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0xE480E480u));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0xE480E480u));
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(x));
    }
}
// Codes 0 and 1 of x beside those of y, as pairs (x0, y0) and (x1, y1); SECOND: codes 2 and 3.
template <int KIND, bool SECOND> __device__ __forceinline__ void beside(unsigned x, unsigned y, unsigned& lo, unsigned& hi) {
    if constexpr (KIND == CACHE_INT8) four<KIND>(__byte_perm(x, y, SECOND ? 0x7632 : 0x5410), lo, hi);
    else four<KIND>(__byte_perm(x, y, SECOND ? 0x7362 : 0x5140), lo, hi);
}

// Exponent field of the power of two that brings a row whose largest magnitude is `top` into [2^13, 2^14), and of its
// reciprocal (254 - field): at least 1, at most 253.
__device__ __forceinline__ int query_field(float top) {
    const int e = (__float_as_int(top) >> 23) & 255;       // (NaN and infinity: 255)
    return min(253, max(1, 127 + 13 + 127 - e));
}
__device__ __forceinline__ float power(int field) { return __int_as_float(field << 23); }

// two bfloat16 times a power of two as float16
__device__ __forceinline__ unsigned half_pair(unsigned two_bf16, float f) {
    const float lo = __uint_as_float(two_bf16 << 16) * f, hi = __uint_as_float(two_bf16 & 0xffff0000u) * f;
    unsigned d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ unsigned half_pair(float lo, float hi) {
    unsigned d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

constexpr float VALUE_FACTOR = 128.f;          // 2^7, see above
// a score whose reference is kept in two numbers, see above (an infinity, whose row has no result, is none)
__device__ __forceinline__ bool coarse_score(float x) { return fabsf(x) >= 16777216.f && fabsf(x) < INFINITY; }
// log2 of a power of two above a value scale, as far as it counts (an infinity or NaN, whose results are none: 0)
__device__ __forceinline__ int scale_log2(float scale) {
    const int e = __float_as_int(scale) >> 23 & 255;
    return e == 255 ? 0 : min(110, max(-100, e - 126));
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace slb_codes
