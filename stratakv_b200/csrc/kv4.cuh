// Keys and values held in 4 bits: how a number is stored and read.
//
// A head's numbers lie in groups of 16.  A group has one scale byte b, which stands for s = half(b << 7) / 64 (the half-precision
// number with those bits: 5 bits of exponent, 3 of mantissa, no sign), and a code of 4 bits per number: code n stands for
// (n - 8) s.  Numbers 2i and 2i + 1 are the low and the high half of byte i.  (n - 8) s has at most 7 significant bits and lies
// between 2^-23 and 6,272, so it is exact in half precision and in bfloat16: what reads the cache rounds nothing.  s is the
// smallest scale with |x| <= 7 s for all of a group (codes 1 to 15); beyond 6,272 a number saturates.  A group that holds an
// infinity or a NaN has scale byte 255, whose half is a NaN, so that it reaches whoever reads it.
#pragma once

#include "common.cuh"

namespace skv {

constexpr int KV4_GROUP = 16;
constexpr uint32_t KV4_LARGEST = 246, KV4_NOT_FINITE = 255;      // (247: 9/8 of its half, which the reading multiplies by, is no half)

__device__ __forceinline__ float kv4_scale(uint32_t byte) {
    return __half2float(__ushort_as_half((unsigned short)(byte << 7))) * 0.015625f;
}

// The scale byte of a group whose largest magnitude is `most` (finite): the smallest with 7 s >= most.
__device__ __forceinline__ uint32_t kv4_scale_byte(float most) {
    const float wanted = __fmul_rn(__fdiv_rn(most, 7.0f), 64.0f);
    // above 2^-14 a half has the float's exponent, 112 less, and the upper 3 bits of its mantissa; below, steps of 2^-17
    uint32_t byte = wanted >= 6.103515625e-05f ? ((__float_as_uint(wanted) + 0xFFFFFu) >> 20) - 896u
                                               : (uint32_t)__float2int_ru(wanted * 131072.0f);
    byte = min(byte, KV4_LARGEST);
    if (7.0f * kv4_scale(byte) < most) ++byte;             // (the quotient was rounded down to a scale; 7 s is exact)
    return min(byte, KV4_LARGEST);
}

// Code of x in a group whose scale has the reciprocal `inverse` (0 where the scale is 0).  Both are rounded to nearest, so that the code
// is the same whoever computes it.
__device__ __forceinline__ uint32_t kv4_code(float x, float inverse) {
    const float steps = fminf(fmaxf(rintf(__fmul_rn(x, inverse)), -7.0f), 7.0f);
    return (uint32_t)((int)steps + 8);
}

// Eight codes as four pairs of half-precision numbers 1 + n / 64: pair p holds codes p and p + 4.  The code lands on bits 4 to 7 of a half's
// mantissa, so that three shifts and four logic operations serve eight numbers.
__device__ __forceinline__ void kv4_spread(uint32_t word, uint32_t (&pairs)[4]) {
    pairs[0] = ((word << 4) & 0x00F000F0u) | 0x3C003C00u;
    pairs[1] = (word & 0x00F000F0u) | 0x3C003C00u;
    pairs[2] = ((word >> 4) & 0x00F000F0u) | 0x3C003C00u;
    pairs[3] = ((word >> 8) & 0x00F000F0u) | 0x3C003C00u;
}

// (n - 8) s of such a pair: (1 + n / 64) h - (9 / 8) h in one multiply-add, exact: s = h / 64, and 9 h / 8 is a half.
__device__ __forceinline__ uint32_t kv4_value(uint32_t pair, uint32_t scale, uint32_t offset) {
    const __half2 v = __hfma2(*(const __half2*)&pair, *(const __half2*)&scale, *(const __half2*)&offset);
    return *(const uint32_t*)&v;
}
// -(9 / 8) h of a pair of scales' halves.
__device__ __forceinline__ uint32_t kv4_offset(uint32_t scale) {
    const __half2 v = __hmul2(*(const __half2*)&scale, __float2half2_rn(-1.125f));
    return *(const uint32_t*)&v;
}

}  // namespace skv
