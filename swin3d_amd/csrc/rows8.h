// Rows in eight bits: what the kernels of norm_int8.hip, linear_int8.hip, kept_rows.hip and the dense layers' gradients share.
//
// Two forms.  For products in whole numbers a row has one fp32 scale, a 127th of its largest number, and codes -127 .. 127.
//
// For what a backward pass reads of a layer's input ("kept" rows) sixteen neighbouring numbers of an fp16 row share a scale of four
// significant bits in units of 2^-24, the smallest with 127 scales reaching the largest of them: a byte with five bits of exponent and
// three of mantissa.  A code of seven bits times such a scale has eleven bits and is a multiple of 2^-24, that is an fp16 number: the
// products of the backward read what a row stands for without another rounding.  What the four bits cost is at most an eighth of a
// step, of which sixteen numbers to a scale, where a whole row has its outliers, give back more (tests/test_gpu_kept_rows.py has both).  At the ends they cost
// more: below 8 2^-24 scales have fewer bits (up to a unit of 2^-24 above a 127th of the largest number), and at the largest scale, 576, codes end at 113,
// that is at 65,088.
#pragma once

#include "dense.h"

namespace s3d {

constexpr int kKeptGroup = 16;
constexpr uint32_t kKeptNaN = 255;      // of a group with a number that is not finite: all of it stands for NaN

// Three bits below five of an exponent, put where fp32 has them, are the scale but for a power of two; below the smallest exponent
// fp32's denormal numbers continue as the scales do.  2^105 = 2^(127 - 22): bits 1 << 20 stand for 2^-129 and mean 2^-24.
__device__ __forceinline__ float kept_step(uint32_t byte) { return __uint_as_float(byte << 20) * 0x1p105f; }
__device__ __forceinline__ float kept_scale(uint32_t byte) { return byte == kKeptNaN ? __builtin_nanf("") : kept_step(byte); }

// The byte of a group's largest size, by its fp16 bits.  Truncated, a / 127 is the scale or the one below, also where the quotient's
// rounding crosses one; 127 times a scale is exact.
__device__ __forceinline__ uint32_t kept_byte(uint32_t largest)
{
    const float a = __builtin_bit_cast(_Float16, static_cast<uint16_t>(largest));
    const uint32_t byte = __float_as_uint(a * (1.0f / 127.0f) * 0x1p-105f) >> 20;
    const uint32_t up = byte + (127.0f * kept_step(byte) < a ? 1 : 0);
    return largest >= 0x7c00u ? kKeptNaN : up;
}

// What turns numbers into codes of a scale.  No branch for the groups that have none: zeros are divided by the smallest scale, and what the
// quotients of a group that is not finite are, NaN included, no code of it is above 0.
struct Divisor {
    float scale, inverse, most;
    __device__ __forceinline__ explicit Divisor(uint32_t byte)
    {
        scale = kept_step(max(byte, 1u));
        inverse = __builtin_amdgcn_rcpf(scale);
        most = byte == kKeptNaN ? 0.0f : byte >= 249 ? 113.0f : 127.0f;      // (114 times the largest scale, 576, would round to infinity in fp16)
    }
    // x / scale to the nearest whole number, ties to even, as the low byte of the result.  The correction makes the quotient the
    // correctly rounded one, with a reciprocal that is a unit off too; without it 2,214 of the 3,981,084 pairs of an fp16 number and a scale
    // that reaches it get the other neighbour of a tie.
    __device__ __forceinline__ uint32_t code(float x) const
    {
        float q = x * inverse;
        q = fmaf(fmaf(-q, scale, x), inverse, q);
        q = __builtin_amdgcn_fmed3f(q, -most, most);
        return __float_as_uint(q + 12582912.0f);      // 1.5 x 2^23: whole numbers lie one unit apart
    }
};

__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// code i of four, as a number
template <int I> __device__ __forceinline__ float code_of(uint32_t four) { return static_cast<float>(static_cast<int>(four << (24 - 8 * I)) >> 24); }

// Eight codes times their scale, in fp16 arithmetic, in which every step is exact: a byte below 0x64 is 1024 + it, less 1152 the code (whose
// sign bit was turned), and that times the scale is an fp16 number.
__device__ __forceinline__ half8 kept_numbers(uint2 codes, uint32_t byte)
{
    const _Float16 s = static_cast<_Float16>(kept_scale(byte)), offset = static_cast<_Float16>(1152.0f);
    const half2 scale = {s, s}, offsets = {offset, offset};
    half8 v;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint32_t four = (w ? codes.y : codes.x) ^ 0x80808080u;
        const half2 lo = (__builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, four, 0x04010400u)) - offsets) * scale;
        const half2 hi = (__builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, four, 0x04030402u)) - offsets) * scale;
        v[4 * w] = lo[0];
        v[4 * w + 1] = lo[1];
        v[4 * w + 2] = hi[0];
        v[4 * w + 3] = hi[1];
    }
    return v;
}

// the largest size among numbers, as fp16 bits, which order infinity and NaN behind all others
typedef uint16_t bits2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b)
{
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(bits2, a), __builtin_bit_cast(bits2, b)));
}
__device__ __forceinline__ uint32_t largest_bits(const half8 &v)
{
    const uint4 w = __builtin_bit_cast(uint4, v);
    const uint32_t pair = larger_pair(larger_pair(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), larger_pair(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(pair >> 16, pair & 0xffffu);
}

__device__ __forceinline__ uint32_t kept_codes(const half4 &v, const Divisor &d) { return four_bytes(d.code(v[0]), d.code(v[1]), d.code(v[2]), d.code(v[3])); }
__device__ __forceinline__ uint2 kept_codes(const half8 &v, const Divisor &d)
{
    return make_uint2(four_bytes(d.code(v[0]), d.code(v[1]), d.code(v[2]), d.code(v[3])),
                      four_bytes(d.code(v[4]), d.code(v[5]), d.code(v[6]), d.code(v[7])));
}

// fp32 first, then fp16: where the compiler makes one instruction of the last operation and the conversion, as it does in some kernels and
// not in others, a number in some 70,000 is the other neighbour of a tie
__device__ __forceinline__ _Float16 to_half(float v)
{
    asm volatile("" : "+v"(v));
    return static_cast<_Float16>(v);
}

// The sums over a product's 32 rows of what its lanes hold in fp32, row lane % 32 and columns 8 g + 4 half + e as v[4 g + e]: in every lane that of column
// summed_column(lane).  Lanes trade half of their numbers for the partner's other half, so that 16 numbers a lane are 38 instructions, where all in
// all lanes would be 96.
template <int kControl> __device__ __forceinline__ float from_lane(float v)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), kControl, 0xf, 0xf, true));
}
template <int kControl, int N> __device__ __forceinline__ void traded(float *v, bool upper)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float own = upper ? v[i + N] : v[i], other = upper ? v[i] : v[i + N];
        v[i] = own + from_lane<kControl>(other);
    }
}
__device__ __forceinline__ float column_sum(float (&v)[16], int lane)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 8]), false, false);
        v[i] = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
    traded<0x128, 4>(v, lane & 8);      // lanes 8 apart, then mirrored ones of eight, then two apart
    traded<0x141, 2>(v, lane & 4);
    traded<0x4e, 1>(v, lane & 2);
    return v[0] + from_lane<0xb1>(v[0]);
}
__device__ __forceinline__ int summed_column(int lane)
{
    const int i = (lane & 31) >> 1;
    return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
}

// x Phi(x) and its derivative at once, of numbers that are finite or NaN: in the terms of gelu_slope, u phi(u) M(u) is what x Phi(x)
// is below the larger of x and 0.
struct Active {
    float value, slope;
};
__device__ __forceinline__ Active gelu_and_slope(float x)
{
    const GeluTail t = gelu_tail(x);
    return {fmaf(-t.u * t.phi, t.u - t.q, fmaxf(x, 0.0f)), fmaf(__builtin_copysignf(t.phi, x), t.q, 0.5f + __builtin_copysignf(0.5f, x))};
}

}  // namespace s3d
