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
    const float wanted = most * 9.142857f;                 // 64 most / 7, nearly
    // above 2^-14 a half has the float's exponent, 112 less, and the upper 3 bits of its mantissa; below, steps of 2^-17
    uint32_t byte = wanted >= 6.103515625e-05f ? ((__float_as_uint(wanted) + 0xFFFFFu) >> 20) - 896u
                                               : (uint32_t)__float2int_ru(wanted * 131072.0f);
    byte = min(byte, KV4_LARGEST);
    // what the factor's and the product's roundings made of it, at most a step either way (7 s is exact)
    if (7.0f * kv4_scale(byte) < most) return min(byte + 1u, KV4_LARGEST);
    return byte && 7.0f * kv4_scale(byte - 1u) >= most ? byte - 1u : byte;
}

// Code of x in a group whose scale has the reciprocal `inverse` (0 where the scale is 0).  Both are rounded to nearest, so that the code is the same
// whoever computes it; adding 1.5 x 2^23 + 8 rounds the quotient to an integer, ties to even, and leaves it + 8 in the lowest bits.
__device__ __forceinline__ uint32_t kv4_code(float x, float inverse) {
    return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x, inverse), -7.0f), 7.0f), 12582920.0f)) & 15u;
}

// Eight codes as four pairs of halves (n - 8) s, exact; pair p holds codes p and p + 4.  A code is brought to bits 4 to 7 of a mantissa, as 1 + n / 64: one
// multiply-add, (1 + n / 64) h - (9 / 8) h, does the rest (h = 64 s; 9 h / 8 is a half).
struct Kv4Scale {
    uint32_t h, offset;                                    // pairs of h and -(9 / 8) h
};
__device__ __forceinline__ Kv4Scale kv4_pair_of_scales(uint32_t h) {
    uint32_t offset;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(offset) : "r"(h), "r"(0xBC80BC80u));
    return {h, offset};
}
// `ones`: the half 1 twice, 0x3C003C00.  It reaches a kernel as an argument: a logic operation takes one constant, and of two that it knows the
// compiler makes two operations (1 x 131,072 positions 45.8 us so, 41.8 with one).
constexpr uint32_t KV4_ONES = 0x3C003C00u;
__device__ __forceinline__ uint32_t kv4_value(uint32_t codes, const Kv4Scale& of, uint32_t ones) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"((codes & 0x00F000F0u) | ones), "r"(of.h), "r"(of.offset));
    return d;
}
__device__ __forceinline__ void kv4_unpack(uint32_t word, const Kv4Scale& of, uint32_t ones, uint32_t (&pairs)[4]) {
    pairs[0] = kv4_value(word << 4, of, ones);
    pairs[1] = kv4_value(word, of, ones);
    pairs[2] = kv4_value(word >> 4, of, ones);
    pairs[3] = kv4_value(word >> 8, of, ones);
}

}  // namespace skv
