// Rows in eight bits with a scale each (gfx950): LayerNorm or root-mean-square norm of x + residual, or rows as they are.
//
//   s = x + residual;  y = (s - mean) / sqrt(var + eps) * gamma + beta   or   s / sqrt(mean(s^2) + eps) * gamma   or   x
//   scale = max |y| / 127;  code = 127 y / max |y| to the nearest whole number, ties to even
//
// All arithmetic in fp32, y without a rounding of its own between norm and code.  A row of zeros has scale 0 and codes 0; one with a
// number that is not finite has codes 0 and scale NaN, so that all that is computed from it is NaN.
//
// Bound by memory: 4 C (+ 2 C or 4 C) bytes in, C + 4 (+ 4 C for the sum) out per row.  A row stays in registers from its loads to its
// codes: up to 1024 channels on G lanes of a wavefront, beyond that on a workgroup, whose sums meet in LDS.  199,327 rows of 48 with an fp16
// residual 19.2 us, 5.5 TB/s, 149,993 of 160 with an fp32 one 55.8, 5.6; 811 of 384 3.7, a launch.
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

constexpr int kThreads = 256;
constexpr int kMostChannels = 8192;

template <int kControl> __device__ __forceinline__ uint32_t moved(uint32_t v)
{
    return __builtin_amdgcn_update_dpp(0u, v, kControl, 0xf, 0xf, true);
}

// Sum or maximum over G lanes, or over a workgroup (G = 256, `shared` of four numbers), in all of them
template <int G, typename T, typename Op> __device__ __forceinline__ T over_lanes(T v, Op op, T *shared)
{
    static_assert(G == 8 || G == 16 || G == 32 || G == 64 || G == kThreads, "rows of a wavefront's lanes, or of all four wavefronts");
    auto bits = [](T x) { return __builtin_bit_cast(uint32_t, x); };
    auto value = [](uint32_t x) { return __builtin_bit_cast(T, x); };
    v = op(v, value(moved<0xb1>(bits(v))));
    v = op(v, value(moved<0x4e>(bits(v))));
    v = op(v, value(moved<0x141>(bits(v))));
    if (G >= 16) v = op(v, value(moved<0x140>(bits(v))));
    if (G >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
        v = op(value(a[0]), value(a[1]));
    }
    if (G >= 64) {
        const auto a = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
        v = op(value(a[0]), value(a[1]));
    }
    if (G > 64) {
        __syncthreads();      // (the last use of `shared`)
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
        __syncthreads();
        v = op(op(shared[0], shared[1]), op(shared[2], shared[3]));
    }
    return v;
}

enum Norm { kNone = 0, kLayer = 1, kRms = 2 };

struct RowArgs {
    const void *x, *residual;       // [N,C] fp32 (kNone: fp32 or fp16), [N,C] or null
    const float *gamma, *beta;      // [C]; null: ones, zeros
    float *sum;                     // [N,C] or null
    int8_t *codes;                  // [N,C]
    float *scales;                  // [N]
    int64_t N;
    int32_t C;
    float eps;
};

template <bool kHalf> __device__ __forceinline__ float4 four_at(const void *from, int64_t at)
{
    if (!kHalf) return *reinterpret_cast<const float4 *>(static_cast<const float *>(from) + at);
    const half4 h = *reinterpret_cast<const half4 *>(static_cast<const _Float16 *>(from) + at);
    return make_float4(h[0], h[1], h[2], h[3]);
}

// RES: 0 none, 1 fp32, 2 fp16.  FOURS: of a lane.
template <int G, int FOURS, int NORM, bool HALF, int RES>
__global__ __launch_bounds__(kThreads) void rows_int8_kernel(RowArgs a)
{
    __shared__ uint32_t shared[4];
    const int lane = threadIdx.x % G, C = a.C, fours = C / 4;
    float *shared_sum = reinterpret_cast<float *>(shared);
    auto add = [](float p, float q) { return p + q; };
    auto larger = [](uint32_t p, uint32_t q) { return max(p, q); };
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G; row < a.N; row += step) {
        float4 v[FOURS], r[FOURS], g[FOURS], b[FOURS];
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            const int at = 4 * min(lane + i * G, fours - 1);
            v[i] = four_at<HALF>(a.x, row * C + at);
            if (RES) r[i] = four_at<RES == 2>(a.residual, row * C + at);
        }
        if (NORM) {
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                const int at = 4 * min(lane + i * G, fours - 1);
                g[i] = a.gamma ? *reinterpret_cast<const float4 *>(a.gamma + at) : make_float4(1, 1, 1, 1);
                b[i] = a.beta ? *reinterpret_cast<const float4 *>(a.beta + at) : make_float4(0, 0, 0, 0);
            }
        }
        if (RES) {
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                v[i].x += r[i].x; v[i].y += r[i].y; v[i].z += r[i].z; v[i].w += r[i].w;
                if (a.sum && lane + i * G < fours) *reinterpret_cast<float4 *>(a.sum + row * C + 4 * (lane + i * G)) = v[i];
            }
        }
        if (NORM) {
            float mean = 0.0f, sq = 0.0f;
            if (NORM == kLayer) {
#pragma unroll
                for (int i = 0; i < FOURS; ++i)
                    if (lane + i * G < fours) mean += (v[i].x + v[i].y) + (v[i].z + v[i].w);
                mean = over_lanes<G>(mean, add, shared_sum) / static_cast<float>(C);
            }
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                if (NORM == kLayer) { v[i].x -= mean; v[i].y -= mean; v[i].z -= mean; v[i].w -= mean; }
                if (lane + i * G < fours) sq += (v[i].x * v[i].x + v[i].y * v[i].y) + (v[i].z * v[i].z + v[i].w * v[i].w);
            }
            const float rstd = 1.0f / sqrtf(over_lanes<G>(sq, add, shared_sum) / static_cast<float>(C) + a.eps);
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                v[i].x = v[i].x * rstd * g[i].x + b[i].x;
                v[i].y = v[i].y * rstd * g[i].y + b[i].y;
                v[i].z = v[i].z * rstd * g[i].z + b[i].z;
                v[i].w = v[i].w * rstd * g[i].w + b[i].w;
            }
        }
        uint32_t most = 0;      // sizes as bits, which order infinity and NaN behind all others
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            auto size = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
            // (a lane without a four has the last one, or the sum that another wavefront has put in its place)
            if (lane + i * G < fours) most = max(max(max(size(v[i].x), size(v[i].y)), max(size(v[i].z), size(v[i].w))), most);
        }
        most = over_lanes<G>(most, larger, shared);
        const bool finite = most < 0x7f800000u;
        const float a_max = finite ? __uint_as_float(most) : 0.0f;
        // (127 / a_max stays finite, and a product with it exact enough, for the smallest rows too)
        const float lift = a_max < 0x1p-100f ? 0x1p100f : 1.0f, inverse = a_max > 0.0f ? 127.0f / (a_max * lift) : 0.0f;
        const float reciprocal = HALF && a_max > 0.0f ? 1.0f / a_max : 0.0f;
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            if (lane + i * G >= fours) continue;
            // Rows of fp16 numbers have ties: where the largest is 127 / 2^n of another number, one number in some twenty lies between two
            // codes exactly.  Their quotient 127 x / a_max is the correctly rounded one (127 x is exact), so that these go to even.
            auto code = [&](float x) {
                if (!HALF) return __float_as_uint(fmaf(finite ? x * lift : 0.0f, inverse, 12582912.0f));
                const float q = x * inverse;
                return __float_as_uint(finite ? fmaf(fmaf(-q, a_max, 127.0f * x), reciprocal, q) + 12582912.0f : 0.0f);
            };
            *reinterpret_cast<uint32_t *>(a.codes + row * C + 4 * (lane + i * G)) = four_bytes(code(v[i].x), code(v[i].y), code(v[i].z), code(v[i].w));
        }
        if (lane == 0) a.scales[row] = finite ? a_max / 127.0f : __builtin_nanf("");
    }
}

template <int G, int FOURS, int NORM, bool HALF, int RES> int launch_rows(const RowArgs &a, hipStream_t stream)
{
    const int64_t blocks = ceil_div(a.N, kThreads / G);
    hipLaunchKernelGGL((rows_int8_kernel<G, FOURS, NORM, HALF, RES>), dim3(static_cast<unsigned>(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(kThreads), 0,
                       stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

template <int NORM, bool HALF, int RES> int launch_width(const RowArgs &a, hipStream_t stream)
{
    const int fours = a.C / 4;
    if (fours <= 16) return launch_rows<16, 1, NORM, HALF, RES>(a, stream);
    if (fours <= 32) return launch_rows<32, 1, NORM, HALF, RES>(a, stream);
    if (fours <= 64) return launch_rows<64, 1, NORM, HALF, RES>(a, stream);
    if (fours <= 128) return launch_rows<64, 2, NORM, HALF, RES>(a, stream);
    if (fours <= 256) return launch_rows<64, 4, NORM, HALF, RES>(a, stream);
    if (fours <= 512) return launch_rows<256, 2, NORM, HALF, RES>(a, stream);
    if (fours <= 1024) return launch_rows<256, 4, NORM, HALF, RES>(a, stream);
    return launch_rows<256, 8, NORM, HALF, RES>(a, stream);
}

template <int NORM> int launch_residual(const RowArgs &a, int res, hipStream_t stream)
{
    if (res == 0) return launch_width<NORM, false, 0>(a, stream);
    return res == 1 ? launch_width<NORM, false, 1>(a, stream) : launch_width<NORM, false, 2>(a, stream);
}

// Rows of fp16 as they are, eight numbers at a time: what is left to do a number is little, so that what counts is bytes a load and lanes without
// any.  Over four numbers at a time: 49.6 / 33.1 us at 595,677 rows of 80, 26.3 / 15.0 at 149,993 of 160 (4.8 TB/s), 31.7 / 22.7 at 37,499 of 1280,
// 10.0 / 8.2 at 199,327 of 48 (12.7 with sixteen lanes a row, ten of them idle), the same within 5% for a few thousand rows and at 4096 channels.
template <int G, int EIGHTS>
__global__ __launch_bounds__(kThreads) void half_rows_int8_kernel(RowArgs a)
{
    const int lane = threadIdx.x % G, C = a.C, eights = C / 8;
    const _Float16 *x = static_cast<const _Float16 *>(a.x);
    auto larger = [](uint32_t p, uint32_t q) { return max(p, q); };
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G; row < a.N; row += step) {
        half8 v[EIGHTS];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < EIGHTS; ++i) v[i] = *reinterpret_cast<const half8 *>(x + row * C + 8 * min(lane + i * G, eights - 1));
#pragma unroll
        for (int i = 0; i < EIGHTS; ++i) most = max(most, largest_bits(v[i]));      // (a lane without an eight has the last one)
        most = over_lanes<G>(most, larger, static_cast<uint32_t *>(nullptr));
        const bool finite = most < 0x7c00u;
        const float a_max = finite ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(most))) : 0.0f;
        const float reciprocal = a_max > 0.0f ? 1.0f / a_max : 0.0f, inverse = a_max > 0.0f ? 127.0f / a_max : 0.0f;
        // 127 x / a_max correctly rounded, so that ties, which rows of fp16 numbers have, go to even
        auto code = [&](float number) {
            const float q = number * inverse;
            return __float_as_uint(finite ? fmaf(fmaf(-q, a_max, 127.0f * number), reciprocal, q) + 12582912.0f : 0.0f);
        };
#pragma unroll
        for (int i = 0; i < EIGHTS; ++i) {
            if (lane + i * G >= eights) continue;
            *reinterpret_cast<uint2 *>(a.codes + row * C + 8 * (lane + i * G)) =
                make_uint2(four_bytes(code(v[i][0]), code(v[i][1]), code(v[i][2]), code(v[i][3])), four_bytes(code(v[i][4]), code(v[i][5]), code(v[i][6]), code(v[i][7])));
        }
        if (lane == 0) a.scales[row] = finite ? a_max / 127.0f : __builtin_nanf("");
    }
}

template <int G, int EIGHTS> int launch_half_rows(const RowArgs &a, hipStream_t stream)
{
    const int64_t blocks = ceil_div(a.N, kThreads / G);
    hipLaunchKernelGGL((half_rows_int8_kernel<G, EIGHTS>), dim3(static_cast<unsigned>(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(kThreads), 0, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

int launch_half(const RowArgs &a, hipStream_t stream)
{
    const int eights = a.C / 8;
    if (eights <= 8) return launch_half_rows<8, 1>(a, stream);
    if (eights <= 16) return launch_half_rows<16, 1>(a, stream);
    if (eights <= 32) return launch_half_rows<16, 2>(a, stream);
    if (eights <= 48) return launch_half_rows<16, 3>(a, stream);
    if (eights <= 64) return launch_half_rows<16, 4>(a, stream);
    if (eights <= 96) return launch_half_rows<32, 3>(a, stream);
    if (eights <= 128) return launch_half_rows<32, 4>(a, stream);
    if (eights <= 192) return launch_half_rows<64, 3>(a, stream);
    if (eights <= 256) return launch_half_rows<64, 4>(a, stream);
    if (eights <= 320) return launch_half_rows<64, 5>(a, stream);
    return launch_half_rows<64, 8>(a, stream);
}

// four numbers a thread (bound by memory: 149,993 rows of 160 to fp16 15.4 us, 4.7 TB/s)
template <bool HALF>
__global__ __launch_bounds__(kThreads) void values_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales, void *out, int64_t total, int fours)
{
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const uint32_t four = reinterpret_cast<const uint32_t *>(codes)[i];
        const float s = scales[i / fours];
        const float4 v = make_float4(code_of<0>(four) * s, code_of<1>(four) * s, code_of<2>(four) * s, code_of<3>(four) * s);
        if (HALF)
            reinterpret_cast<half4 *>(out)[i] = half4{static_cast<_Float16>(v.x), static_cast<_Float16>(v.y), static_cast<_Float16>(v.z), static_cast<_Float16>(v.w)};
        else
            reinterpret_cast<float4 *>(out)[i] = v;
    }
}

bool fits(int64_t N, int32_t C) { return N >= 0 && N <= 0x7fffffff && C >= 4 && C % 4 == 0 && C <= kMostChannels; }
int bad_shape(const char *who, int64_t N, int32_t C)
{
    return fail(S3D_ERR_BAD_SHAPE, "%s: N=%lld C=%d (C a multiple of 4, 4..%d)", who, (long long)N, C, kMostChannels);
}

}  // namespace

int launch_quantize_rows(const void *x, int32_t dtype, int8_t *codes, float *scales, int64_t N, int32_t C, hipStream_t stream)
{
    const RowArgs a{x, nullptr, nullptr, nullptr, nullptr, codes, scales, N, C, 0.0f};
    if (dtype == S3D_DTYPE_F16 && C % 8 == 0 && C <= 4096) return launch_half(a, stream);
    return dtype == S3D_DTYPE_F16 ? launch_width<kNone, true, 0>(a, stream) : launch_width<kNone, false, 0>(a, stream);
}

}  // namespace s3d

extern "C" __attribute__((visibility("default"))) int s3d_add_norm_int8(
    const float *x, const void *residual, int32_t residual_dtype, const float *gamma, const float *beta, float eps, int32_t rms, float *sum,
    int8_t *codes, float *scales, int64_t N, int32_t C, void *stream)
{
    using namespace s3d;
    if (!fits(N, C)) return bad_shape("s3d_add_norm_int8", N, C);
    if (residual && residual_dtype != S3D_DTYPE_F32 && residual_dtype != S3D_DTYPE_F16)
        return fail(S3D_ERR_BAD_DTYPE, "s3d_add_norm_int8: residual_dtype %d (0 = fp32, 1 = fp16)", residual_dtype);
    if (N == 0) return S3D_OK;
    if (!x || !codes || !scales) return fail(S3D_ERR_NULL_POINTER, "s3d_add_norm_int8: null device pointer");
    const RowArgs a{x, residual, gamma, beta, residual ? sum : nullptr, codes, scales, N, C, eps};
    const int res = !residual ? 0 : residual_dtype == S3D_DTYPE_F32 ? 1 : 2;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return rms ? launch_residual<kRms>(a, res, s) : launch_residual<kLayer>(a, res, s);
}

extern "C" __attribute__((visibility("default"))) int s3d_quantize_rows(const void *x, int32_t dtype, int8_t *codes, float *scales, int64_t N, int32_t C,
                                                                        void *stream)
{
    using namespace s3d;
    if (!fits(N, C)) return bad_shape("s3d_quantize_rows", N, C);
    if (dtype != S3D_DTYPE_F32 && dtype != S3D_DTYPE_F16) return fail(S3D_ERR_BAD_DTYPE, "s3d_quantize_rows: dtype %d (0 = fp32, 1 = fp16)", dtype);
    if (N == 0) return S3D_OK;
    if (!x || !codes || !scales) return fail(S3D_ERR_NULL_POINTER, "s3d_quantize_rows: null device pointer");
    return launch_quantize_rows(x, dtype, codes, scales, N, C, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) int s3d_int8_values(const int8_t *codes, const float *scales, void *out, int32_t dtype, int64_t N, int32_t C,
                                                                      void *stream)
{
    using namespace s3d;
    if (!fits(N, C)) return bad_shape("s3d_int8_values", N, C);
    if (dtype != S3D_DTYPE_F32 && dtype != S3D_DTYPE_F16) return fail(S3D_ERR_BAD_DTYPE, "s3d_int8_values: dtype %d (0 = fp32, 1 = fp16)", dtype);
    if (N == 0) return S3D_OK;
    if (!codes || !scales || !out) return fail(S3D_ERR_NULL_POINTER, "s3d_int8_values: null device pointer");
    const int64_t total = N * (C / 4), blocks = ceil_div(total, kThreads);
    auto kernel = dtype == S3D_DTYPE_F16 ? values_kernel<true> : values_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), codes,
                       scales, out, total, C / 4);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}
