// Keys and values in 4 bits: what a byte stands for, and how numbers become bytes.
//
// 16 consecutive elements of a head of one token are a group.  A group has one scale s, held as a byte b that is the upper part of
// the half s / 8: s = 8 half(b << 7), 5 bits of exponent and 3 of fraction, no sign (from 2^-11 on four significant bits, below that
// the multiples of 2^-14).  An element is a whole number c of [-7, 7], held as c + 8 in 4 bits, element 2i in the low half of byte i.
// The value is c s: 4.5 bits an element.
//   s = the number nearest to min(max |x|, 3360) / 7 that a byte can be (at most 480), c = the whole number nearest to x / s, ties to even.
// A group with an element that is not finite has b = 0xff, a NaN, and all its elements read as NaN: as with a cache of 16 bits, what
// is wrong in a token reaches every row that sees the token, and no other.
//
// Why these numbers.  c s has at most 3 + 4 significant bits: it is exact in bfloat16, and c s / 8 in half, so the kernels that put
// codes back into operands of the tensor cores round nothing.  s / 8 stays below 63.5 so that the constant 1032 (s / 8) of that
// conversion is finite in half (see Words in attention4.cu).  A scale for 16 elements costs half a bit an element; per 32 elements
// with 16 bits it would cost the same and leave a larger step (2.1 against 2.4 standard deviations to the largest of a group).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace citlali {
namespace c4 {

constexpr int kGroup = 16;
constexpr float kUnit = 8.0f;
constexpr float kLargestScale = 480.0f;
constexpr int kNoNumber = 0xff;

// |x| as a whole number: in the order of the magnitudes, infinities and then NaNs last (fmaxf would lose a NaN).
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// x / d, rounded to nearest: a product with the reciprocal, off by a last place or two, and one step from the exact remainder.  (Half
// of what the division of all floats takes; the quotients here are far from the ends of the range.)  In particular a quotient that is
// a float comes out as that: a tie between two codes is one.
__device__ __forceinline__ float quotient(float x, float d, float reciprocal) {
    const float q = x * reciprocal;
    return fmaf(fmaf(-q, d, x), reciprocal, q);
}

// The scale's byte for a group whose largest magnitude is `most`, and the scale.
__device__ __forceinline__ int scale_byte(uint32_t most, float& s) {
    if (most >= 0x7f800000u) {
        s = __int_as_float(0x7fc00000);
        return kNoNumber;
    }
    const float wanted = fminf(quotient(fminf(__uint_as_float(most), 7.0f * kLargestScale), 7.0f, 1.0f / 7.0f), kLargestScale);
    if (wanted < 0.00048828125f) {                                   // below 2^-11: multiples of 2^-14
        const float n = rintf(wanted * 16384.0f);
        s = n * 0.00006103515625f;
        return (int)n;
    }
    uint32_t bits = __float_as_uint(wanted);
    bits = (bits + 0x7ffffu + ((bits >> 20) & 1u)) & 0xfff00000u;    // three bits of fraction, ties to even
    s = __uint_as_float(bits);
    return (int)(((bits >> 23) - 127u + 12u) << 3 | ((bits >> 20) & 7u));
}

// Eight elements' codes c + 8 as a word, the first element's in the lowest bits.  1.5 2^23 + 8 + c, added up in a float, rounds to the
// nearest c, ties to even, and has c + 8 in its lowest bits: so one multiply-add a code puts the word together.  A group that holds no
// number, or zeros alone, gets codes that mean nothing, or zeros.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float s) {
    const bool some = s > 0.0f;
    const float d = some ? s : 0.0f, reciprocal = some ? __frcp_rn(s) : 0.0f;
    constexpr uint32_t kOne = 0x4b400000u;                           // the bits of 1.5 2^23
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float c = fminf(fmaxf(quotient(x[i], d, reciprocal), -7.0f), 7.0f);
        w = w * 16u + (__float_as_uint(c + 12582920.0f) - kOne);
    }
    return w;
}

__device__ __forceinline__ float scale_of(uint32_t byte) {
    return __half2float(__ushort_as_half((unsigned short)(byte << 7))) * kUnit;
}

// A word's eight values in bfloat16, two a word, in order.  (w & 0x000f000f) | 0x4300 is 136 + c there, and (136 + c) s - 136 s is
// exact: s has four significant bits, 136 s eight at most.
__device__ __forceinline__ void values_of(uint32_t w, float s, uint32_t (&out)[4]) {
    const __nv_bfloat162 s2 = __float2bfloat162_rn(s), low = __float2bfloat162_rn(-136.0f * s);
    uint32_t pair[4];                                                // elements (i, i + 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t x = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&x), s2, low);
        pair[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    out[0] = __byte_perm(pair[0], pair[1], 0x5410);
    out[1] = __byte_perm(pair[2], pair[3], 0x5410);
    out[2] = __byte_perm(pair[0], pair[1], 0x7632);
    out[3] = __byte_perm(pair[2], pair[3], 0x7632);
}

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_word(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// A scale (or two keys' scales) as the conversion needs it.
struct Scale {
    __half2 s, low, high;                                // s, -1032 s, -72 s
    __device__ __forceinline__ explicit Scale(uint32_t two_bytes) {      // bytes 0 and 2
        s = as_half2(two_bytes << 7);
        low = __hmul2(s, __float2half2_rn(-1032.0f));
        high = __hmul2(s, __float2half2_rn(-72.0f));
    }
};
// (w & mask) | bits in one instruction: written in C it becomes two, since only one of two constants fits an instruction.
template <uint32_t kMask>
__device__ __forceinline__ __half2 picked(uint32_t w, uint32_t bits) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w), "n"(kMask), "r"(bits));
    return as_half2(x);
}
// Nibbles 0 and 4 (first), 1 and 5 (second) of a word times the scale.  The two constants stay in registers.
struct Words {
    uint32_t low, high;
    __device__ __forceinline__ Words() {
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(low));
        asm volatile("mov.b32 %0, 0x54005400;" : "=r"(high));
    }
    __device__ __forceinline__ uint32_t first_of(uint32_t w, const Scale& k) const { return as_word(__hfma2(picked<0x000f000fu>(w, low), k.s, k.low)); }
    __device__ __forceinline__ uint32_t second_of(uint32_t w, const Scale& k) const { return as_word(__hfma2(picked<0x00f000f0u>(w, high), k.s, k.high)); }
};

// Where a token's key or value of a head lies: codes [page][head][token of the page][d / 2], scales [page][head][token][d / 16].
__device__ __forceinline__ size_t place(int page, int nkv, int head, int page_size, int at) {
    return ((size_t)page * nkv + head) * page_size + at;             // times d / 2 or d / 16
}

}  // namespace c4
}  // namespace citlali
