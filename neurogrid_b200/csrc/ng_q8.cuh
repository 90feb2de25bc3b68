// Keys and values held in 8 bits: the codes (e4m3, or integers -127..127) and the scale of a block of tokens and head.
//
// A code c stands for c * scale; scales are powers of two.  Both kinds of codes are exact in float16 (e4m3: four significant bits,
// 2^-9 .. 448; integers: seven bits), so the tensor cores can take the codes themselves as float16 operands, and a scale, being the
// same for a block, is applied to the 32-bit scores and weights.  A power of two loses nothing of e4m3's relative precision, makes a
// value code * scale exact in bfloat16 and float32, and lets a block's scale grow while e4m3 codes that were there keep their bits
// (but for those that fall below its smallest normal number).  Integers lose at most a bit of the block's range to it.
#pragma once
#include "ng_common.cuh"

enum { NG_Q8_E4M3 = 0, NG_Q8_INT8 = 1 };
#define NG_Q8_EXP_LOWEST (-100)
#define NG_Q8_EXP_HIGHEST 100

// four codes -> four float16 (two words, codes 0,1 and 2,3)
template <int KIND>
__device__ __forceinline__ void q8_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (KIND == NG_Q8_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // 0x64uu is the float16 1024 + uu: the code plus 128 as uu, then less 1152
        const uint32_t u = w ^ 0x80808080u, off = 0x64806480u;
        lo = __byte_perm(u, 0x64646464u, 0x4140);
        hi = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(off));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(off));
    }
}
// two values, already divided by the scale -> two codes (a in the low byte), to nearest, ties to even, saturated.
// NaN stays NaN in e4m3 and becomes 0 in integers.
template <int KIND>
__device__ __forceinline__ uint32_t q8_from_float(float a, float b) {
    if constexpr (KIND == NG_Q8_E4M3) {
        uint16_t d;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
        return d;
    } else {
        const int x = min(max(__float2int_rn(a), -127), 127), y = min(max(__float2int_rn(b), -127), 127);
        return (uint32_t)(x & 0xff) | (uint32_t)(y & 0xff) << 8;
    }
}
// the exponent of the least power of two with which `top` (finite, >= 0) fits the largest code: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
template <int KIND>
__device__ __forceinline__ int q8_exponent(float top) {
    const uint32_t b = __float_as_uint(top);
    const int e = (int)(b >> 23) - 127 - (KIND == NG_Q8_E4M3 ? 8 : 6) + ((b & 0x7fffffu) > (KIND == NG_Q8_E4M3 ? 0x600000u : 0x7e0000u));
    return min(max(e, NG_Q8_EXP_LOWEST), NG_Q8_EXP_HIGHEST);
}
__device__ __forceinline__ float q8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }       // -126 <= e <= 127
__device__ __forceinline__ int q8_exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23 & 0xff) - 127; }
// log2 of a scale, and its reciprocal, from its bits
__device__ __forceinline__ float q8_log2(float scale) {
    return __uint_as_float(0x4b000000u | __float_as_uint(scale) >> 23) - 8388735.f;        // (2^23 + field) - (2^23 + 127)
}
__device__ __forceinline__ float q8_recip(float scale) { return __uint_as_float((254u << 23) - (__float_as_uint(scale) & 0x7f800000u)); }
