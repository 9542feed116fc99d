// Rows in eight bits: what the kernels of norm_int8.hip, linear_int8.hip, kept_rows.hip and the dense layers' gradients share.
//
// Two forms.  For products in whole numbers a row has one fp32 scale, a 127th of its largest number, and codes -127 .. 127.
//
// For what a backward pass reads of a layer's input ("kept" rows) sixteen neighbouring numbers of an fp16 row share a scale of four
// significant bits in units of 2^-24, the smallest with 127 scales reaching the largest of them: a byte with five bits of exponent and
// three of mantissa.  A code of seven bits times such a scale has eleven bits and is a multiple of 2^-24, that is an fp16 number: the
// products of the backward read what a row stands for without another rounding.  What the four bits cost is at most an eighth of a
// step, of which sixteen numbers to a scale, where a whole row has its outliers, give back more (tests/test_gpu_kept_rows.py has both).
#pragma once

#include "dense.h"

namespace s3d {

constexpr int kKeptGroup = 16;
constexpr uint32_t kKeptNaN = 255;      // of a group with a number that is not finite: all of it stands for NaN

// Three bits below five of an exponent, put where fp32 has them, are the scale but for a power of two; below the smallest exponent
// fp32's denormal numbers continue as the scales do.  2^105 = 2^(127 - 22): bits 1 << 20 stand for 2^-129 and mean 2^-24.
__device__ __forceinline__ float kept_scale(uint32_t byte)
{
    return byte == kKeptNaN ? __builtin_nanf("") : __uint_as_float(byte << 20) * 0x1p105f;
}

// The byte of a group's largest size, given as an fp32 number (that is an fp16 number) by its bits.  Truncated, a / 127 is the scale
// or the one below, also where the quotient's rounding crosses one; 127 times a scale is exact.
__device__ __forceinline__ uint32_t kept_byte(uint32_t largest)
{
    if (largest >= 0x7f800000u) return kKeptNaN;
    const float a = __uint_as_float(largest);
    const uint32_t byte = __float_as_uint(a * (1.0f / 127.0f) * 0x1p-105f) >> 20;
    return byte + (127.0f * kept_scale(byte) < a ? 1 : 0);
}

// What turns numbers into codes of a scale
struct Divisor {
    float scale, inverse, most;
    __device__ __forceinline__ explicit Divisor(uint32_t byte)
    {
        scale = kept_scale(byte);
        const bool none = byte == 0 || byte == kKeptNaN;
        scale = none ? 0.0f : scale;
        inverse = none ? 0.0f : 1.0f / scale;
        most = byte >= 249 ? 113.0f : 127.0f;      // (114 times the largest scale, 576, would round to infinity in fp16)
    }
    // x / scale to the nearest whole number, ties to even, as the low byte of the result.  The correction makes the quotient the
    // correctly rounded one, without which 2,214 of the 3,981,084 pairs of an fp16 number and a scale that reaches it get the other
    // neighbour of a tie.
    __device__ __forceinline__ uint32_t code(float x) const
    {
        float q = x * inverse;
        q = fmaf(fmaf(-q, scale, x), inverse, q);
        q = fminf(fmaxf(q, -most), most);
        return __float_as_uint(q + 12582912.0f);      // 1.5 x 2^23: whole numbers lie one unit apart
    }
};

__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// code i of four, as a number
template <int I> __device__ __forceinline__ float code_of(uint32_t four) { return static_cast<float>(static_cast<int>(four << (24 - 8 * I)) >> 24); }

// eight codes times their scale: exact
__device__ __forceinline__ half8 kept_numbers(uint2 codes, uint32_t byte)
{
    const float s = kept_scale(byte);
    half8 v;
    v[0] = static_cast<_Float16>(code_of<0>(codes.x) * s);
    v[1] = static_cast<_Float16>(code_of<1>(codes.x) * s);
    v[2] = static_cast<_Float16>(code_of<2>(codes.x) * s);
    v[3] = static_cast<_Float16>(code_of<3>(codes.x) * s);
    v[4] = static_cast<_Float16>(code_of<0>(codes.y) * s);
    v[5] = static_cast<_Float16>(code_of<1>(codes.y) * s);
    v[6] = static_cast<_Float16>(code_of<2>(codes.y) * s);
    v[7] = static_cast<_Float16>(code_of<3>(codes.y) * s);
    return v;
}

// the largest size among eight numbers, as fp32 bits, which order infinity and NaN behind all others
__device__ __forceinline__ uint32_t largest_bits(const half8 &v)
{
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(static_cast<float>(v[e])) & 0x7fffffffu);
    return most;
}

__device__ __forceinline__ uint2 kept_codes(const half8 &v, const Divisor &d)
{
    return make_uint2(four_bytes(d.code(v[0]), d.code(v[1]), d.code(v[2]), d.code(v[3])),
                      four_bytes(d.code(v[4]), d.code(v[5]), d.code(v[6]), d.code(v[7])));
}

}  // namespace s3d
