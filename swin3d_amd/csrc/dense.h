// Pieces shared by the kernels of the dense layers (linear.hip, mlp.hip).
#pragma once

#include "s3d_common.h"

namespace s3d {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// x Phi(x) = (x + |x|) / 2 - |x| Phi(-|x|), with 2 Phi(-u) = 2^p(u): the logarithm of the normal distribution's tail is
// close to a parabola, and the polynomial of degree 7 with p(0) = 0 that fits it best for |x| Phi(-|x|) over [0, 5.8] (least
// squares at Chebyshev nodes) is 2.5e-7 off, the rounding of fp32; from 5.8 on the tail is below fp16's smallest number.
// Fifteen instruction slots where a rational form with an exponential took 22, and small results keep fp16's relative
// precision.  Infinities and NaN as x Phi(x) has them: the first sum is NaN for -infinity.
__device__ __forceinline__ float gelu(float x)
{
    const float u = fabsf(x), c = fminf(u, 5.8f);
    float p = fmaf(-7.429386528e-7f, c, 4.341329259e-5f);
    p = fmaf(p, c, -8.166006301e-4f);
    p = fmaf(p, c, 8.171264082e-3f);
    p = fmaf(p, c, -5.347365886e-2f);
    p = fmaf(p, c, -4.587851465e-1f);
    p = fmaf(p, c, -1.151172519f);
    return 0.5f * fmaf(-c, __builtin_amdgcn_exp2f(p * c), x + u);
}

// The derivative of x Phi(x): Phi(x) + x phi(x), in fp32.  With Phi(-u) = phi(u) M(u), M the ratio of Mills, that is
// phi(u) (u - M(u)) with the sign of x, and 1 more for x above 0, u = |x|: u - M(u) by the polynomial of degree 12 that fits
// phi(u) (u - M(u)) best over [0, 5.8], 8.7e-9 off at most, up to 5, where phi is still large enough to hold its relative error, and by
// a line from there on, where u - M(u) is close to one.  Over all fp16 numbers the error is the rounding of fp32, 9.2e-8 at most
// (1.47e-7 with erff and the exponential apart).  Where the derivative is small and negative it is a relative 1.4e-4 at most from -3 to
// -5, 1.0e-3 to -8 and 6.5e-3 to -13 (1.7e-3, 3.3e-2 and 2.1e-2, since 1 + erf cancels there; with the polynomial alone 3e-2 at -5.8, and beyond -6.8
// the other sign).  Infinities and NaN as the sum of
// the two terms has them: NaN.  A third of the instructions less: 199,327 rows of 48 to 192, us, 52.6 -> 41.5, 49,682 of 96 to 384
// 33.4 -> 27.0, 12,421 of 192 to 768 24.2 -> 19.0, with their rows alone 18, 15 and 12.
struct GeluTail {
    float u, phi, q;      // |x|, phi(u), u - M(u)
};
__device__ __forceinline__ GeluTail gelu_tail(float x)
{
    const float u = fabsf(x), c = fminf(u, 5.0f), phi = __builtin_amdgcn_exp2f(fmaf(u * u, -0.7213475204f, -1.325748064f));
    float q = fmaf(-1.467262933e-07f, c, 4.019878816e-06f);
    q = fmaf(q, c, -4.986505519e-05f);
    q = fmaf(q, c, 3.754729696e-04f);
    q = fmaf(q, c, -1.954356674e-03f);
    q = fmaf(q, c, 7.658625022e-03f);
    q = fmaf(q, c, -2.421350777e-02f);
    q = fmaf(q, c, 6.534569710e-02f);
    q = fmaf(q, c, -1.560686380e-01f);
    q = fmaf(q, c, 3.331732452e-01f);
    q = fmaf(q, c, -6.266347766e-01f);
    q = fmaf(q, c, 1.999998808e+00f);
    q = fmaf(q, c, -1.253314137e+00f);
    return {u, phi, fmaf(u - c, 1.025f, q)};
}
__device__ __forceinline__ float gelu_slope(float x)
{
    const GeluTail t = gelu_tail(x);
    return fmaf(__builtin_copysignf(t.phi, x), t.q, 0.5f + __builtin_copysignf(0.5f, x));
}

// between what a wavefront's lanes write to its LDS and what other lanes of it read (it serves a wavefront in order)
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr int kPieces = 8;      // of 16 bytes: what is staged of a row of the operands at a time

// The place of 16-byte piece p of row r: sixteen consecutive rows' pieces p lie in 64 different banks.
__device__ __forceinline__ int placed(int r, int p) { return r * kPieces + (p ^ ((r >> 1) & (kPieces - 1))); }

// Sixteen bytes a lane from `from` to the wavefront's 1024 at `to` in LDS.  The compiler knows nothing of them: who reads them
// has waited for them (loads and stores end in the order of their issue) and met the other wavefronts at a barrier.  (m0 is reserved,
// of which it warns; named, it is a definition of m0, which the compiler's own uses of it have to respect.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(uint32_t to, const void *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}
// ... from `base`, the same for all lanes, and a lane's offset in bytes
__device__ __forceinline__ void load_to_lds_from(uint32_t to, const void *base, uint32_t offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "m0", "memory");
}
#pragma clang diagnostic pop
// ... all but the kBehind instructions issued last
template <int kBehind> __device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kBehind) : "memory"); }
__device__ __forceinline__ void workgroup_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace s3d
