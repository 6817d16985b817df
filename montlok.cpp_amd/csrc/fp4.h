// Four-bit values in groups of 32 with a common power of two (OCP MX: e2m1
// codes, an e8m0 scale byte), as the cache and the weights hold them.
//
//   value = (-1)^(code >> 3) * {0, 0.5, 1, 1.5, 2, 3, 4, 6}[code & 7] * 2^(byte - 127);  byte 255: NaN
//
// A value has two significant bits, so up to byte 252 every one of them is exact
// in bf16 and its product with a bf16 number is exact in fp32: sums over it on
// the bf16 matrix cores round only in their fp32 accumulation. Under bytes 253
// and 254 the larger codes stand for 2^128 and more, infinities in bf16; the
// package's own quantisation ends at 252. The conversions are gfx950's
// v_cvt_scalef32_pk_*: over all 256 bytes and all codes they give the values
// above (infinities from 2^128 on, NaN for 255, 2^-127 for byte 0), and the way
// back rounds to nearest with ties to the even code and saturates at 6 (49,160
// values on and next to every border, at 8 scales).
#pragma once

#include "mlk_common.h"

namespace mlk {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // at any element's alignment

constexpr int kGroup = 32;  // values under one scale
constexpr uint32_t kMostScale = 252;  // the largest byte whose values are all finite in bf16 (6 * 2^126 is 1.5 * 2^128)

// The float whose exponent bits are the scale byte: what the conversions take as scale.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Byte `i` of a dword as a scale: shifted to the exponent's place. The neighbouring bits that come along as sign and
// significand do not count (all bytes and codes, 64 patterns of them each, convert alike).
template <int i>
__device__ __forceinline__ float scale_at(uint32_t dword) {
    if constexpr (i == 3) return __uint_as_float(dword >> 1);
    return __uint_as_float(dword << ((23 - 8 * i) & 31));
}

template <int byte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, byte));
}

// Eight codes (low four bits first) under one scale.
__device__ __forceinline__ bf16x8 fp4_octet(uint32_t codes, float scale) {
    const u32x4 v = {fp4_pair<0>(codes, scale), fp4_pair<1>(codes, scale), fp4_pair<2>(codes, scale), fp4_pair<3>(codes, scale)};
    return __builtin_bit_cast(bf16x8, v);
}

// The scale byte of a group whose largest magnitude is `most` (finite): the smallest power of two with
// most <= 6 * 2^(byte - 127). 6 is 1.5 * 2^2, so that is the exponent of `most` less 2, or less 1 where its
// significand is above 1.5. Held to [3, 252]: 6 * 2^125 is finite, 0.5 * 2^-124 normal.
__device__ __forceinline__ uint32_t scale_byte(float most) {
    const int byte = static_cast<int>((__float_as_uint(most) + 0x3FFFFFu) >> 23) - 2;
    return static_cast<uint32_t>(min(max(byte, 3), 252));
}

// An fp32 value as the sum of three bf16 values: its leading 8 significant bits, the next 8, the rest (each cut off, so that
// none of them overflows). Exact from 2^-110 on; below, what is smaller than bf16's least number, 2^-133, is lost. An infinity or a NaN stays alone with CAREFUL, and makes the rest NaN
// without: half the instructions, for callers that look at their result.
struct Parts3 {
    float a, b, c;
};
template <bool CAREFUL>
__device__ __forceinline__ Parts3 parts_of(float x) {
    const uint32_t bits = __float_as_uint(x);
    Parts3 p;
    p.a = __uint_as_float((CAREFUL && x != x ? bits | 0x400000u : bits) & 0xFFFF0000u);
    const float rest = CAREFUL && (bits & 0x7F800000u) == 0x7F800000u ? 0.0f : x - p.a;
    p.b = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
    p.c = rest - p.b;
    return p;
}
// The upper halves of two floats that are bf16 values.
__device__ __forceinline__ uint32_t pack_upper(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// Eight fp32 values as three bf16 operands.
template <bool CAREFUL>
__device__ __forceinline__ void planes_of(const float (&x)[8], bf16x8 (&plane)[3]) {
    u32x4 v[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Parts3 lo = parts_of<CAREFUL>(x[2 * i]), hi = parts_of<CAREFUL>(x[2 * i + 1]);
        v[0][i] = pack_upper(lo.a, hi.a);
        v[1][i] = pack_upper(lo.b, hi.b);
        v[2][i] = pack_upper(lo.c, hi.c);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) plane[i] = __builtin_bit_cast(bf16x8, v[i]);
}

__device__ __forceinline__ float bf16_to_float(uint32_t low16) { return __uint_as_float(low16 << 16); }
// Nearest even; a NaN stays one.
__device__ __forceinline__ uint32_t float_to_bf16(float x) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(x)));
}

// Element access by the tensors' type.
template <bool F32>
struct Element {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};
template <>
struct Element<false> {
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return bf16_to_float(static_cast<const uint16_t*>(p)[i]); }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(float_to_bf16(v)); }
};

}  // namespace mlk
