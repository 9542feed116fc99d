// Y = X W^T + b of rows in eight bits, with GELU on request (gfx950):
//   y[m][n] = sx[m] sw[n] (sum over k of x[m][k] w[n][k]) + b[n]
// x and w whole numbers -127 .. 127, the sum in 32 bits and exact, scales, bias and GELU in fp32, one rounding to fp16.
//
// The plan of linear.hip with bytes in place of fp16 numbers: a chunk is 128 numbers of K of a tile's rows of X and W, in LDS by direct
// loads, and a step of v_mfma_i32_32x32x32_i8 takes 32 of them, sixteen (a piece of 16 bytes) from each half of the lanes.  K is a
// multiple of 16: where half a step is left, the upper lanes put in zeros.
#include "attn_kernels.h"
#include "dense.h"
#include "linear.h"

namespace s3d {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kChunk = 16 * kPieces;      // numbers of K staged at a time

__device__ __forceinline__ i32x16 product(const i32x4 &a, const i32x4 &b, const i32x16 &c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

// WM x WN wavefronts of TM x TN products of 32 x 32
template <int WM, int WN, int TM, int TN> struct Tile {
    static_assert(WM * WN == kThreads / 64, "four wavefronts");
    static constexpr int kWM = WM, kTM = TM, kTN = TN;
    static constexpr int kM = 32 * WM * TM, kN = 32 * WN * TN;
    static constexpr int kStage = (kM + kN) * kChunk;                 // bytes of one staged chunk
    static constexpr int kPitch = 32 * TN + 8;                        // of 32 finished rows of a wavefront
    static_assert(kThreads / 64 * 32 * kPitch * 2 <= kStage, "they fit a buffer");
    static constexpr int kLds = 2 * kStage;
    static constexpr int kLoads = (kM + kN) * kPieces / kThreads;     // pieces per thread and chunk
};

struct Int8Args {
    const int8_t *x, *w;
    const float *sx, *sw, *bias;      // [M], [N], [N] or null
    _Float16 *y;
    int32_t M, N, K, tiles_n, tiles;
};

template <typename L, bool kGelu>
__global__ __launch_bounds__(kThreads, 2) void linear_int8_kernel(Int8Args a)
{
    constexpr int TM = L::kTM, TN = L::kTN;
    __shared__ __align__(16) char smem[L::kLds];
    // workgroups b, b + 8, .. run on one XCD: they get neighbouring tiles, which share rows of X
    const int M = a.M, N = a.N, K = a.K, share = (a.tiles + 7) / 8, begin = static_cast<int>(blockIdx.x) % 8 * share, end = min(begin + share, a.tiles);
    const int step = static_cast<int>(gridDim.x) / 8;
    int tile = begin + static_cast<int>(blockIdx.x) / 8;
    if (tile >= end) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave_m = wave % L::kWM * (32 * TM), wave_n = wave / L::kWM * (32 * TN);
    const int r32 = lane & 31, half = lane >> 5;
    const int whole = (K - 1) / kChunk, left = K - whole * kChunk;      // chunks before the last one, numbers of it

    // This thread's pieces of a chunk: row (tid / 8 + 32 i) of [X rows, W rows], and of it the piece whose place is lane % 8, as
    // sixteen bytes a lane go to consecutive places.  Where the last chunk has no such piece the lane loads its first one.
    const int row = tid / kPieces, piece = (lane ^ (row >> 1)) & (kPieces - 1);
    const int8_t *from[L::kLoads];
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem));
    auto aim = [&](int m0, int n0) {
#pragma unroll
        for (int i = 0; i < L::kLoads; ++i) {
            const int r = row + i * (kThreads / kPieces);
            from[i] = r < L::kM ? a.x + static_cast<int64_t>(min(m0 + r, M - 1)) * K : a.w + static_cast<int64_t>(min(n0 + r - L::kM, N - 1)) * K;
        }
    };
    auto fetch = [&](int buffer, int k0) {
        const int k = k0 + (k0 + piece * 16 < K ? piece * 16 : 0);
#pragma unroll
        for (int i = 0; i < L::kLoads; ++i) load_to_lds(lds + buffer * L::kStage + i * (kThreads * 16) + wave * 1024, from[i] + k);
    };
    i32x16 acc[TM][TN];
    auto multiply = [&](int buffer, int numbers) {
        const i32x4 *at = reinterpret_cast<const i32x4 *>(smem + buffer * L::kStage);
#pragma unroll
        for (int s = 0; s < kChunk / 32; ++s) {
            if (32 * s >= numbers) break;
            i32x4 p[TM], q[TN];
            const bool there = 32 * s + 16 * half < numbers;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                p[i] = at[placed(wave_m + i * 32 + r32, 2 * s + half)];
                p[i] = there ? p[i] : i32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) q[j] = at[placed(L::kM + wave_n + j * 32 + r32, 2 * s + half)];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = product(q[j], p[i], acc[i][j]);
        }
    };
    int buffer = 0;
    bool inside = false;      // the tile before left all its rows and columns: as many stores behind the loads under way
    aim(tile / a.tiles_n * L::kM, tile % a.tiles_n * L::kN);
    fetch(0, 0);
    for (; tile < end; tile += step) {
        const int m0 = tile / a.tiles_n * L::kM, n0 = tile % a.tiles_n * L::kN;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};
        // the chunk is there, and nobody reads the other buffer any more
        auto meet = [&]() {
            if (inside) loads_done<TM * 2 * TN>();
            else loads_done<0>();
            inside = false;
            workgroup_barrier();
        };
        for (int c = 0; c < whole; ++c) {
            meet();
            fetch(buffer ^ 1, (c + 1) * kChunk);
            multiply(buffer, kChunk);
            buffer ^= 1;
        }
        meet();
        // what the end of the tile reads, before the next tile's first chunk: loads return in order
        float4 b[TN][4], sw[TN][4];
        float sx[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) sx[i] = a.sx[min(m0 + wave_m + i * 32 + r32, M - 1)];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = min(n0 + wave_n + j * 32 + 8 * g + 4 * half, N - 4);
                sw[j][g] = *reinterpret_cast<const float4 *>(a.sw + n);
                b[j][g] = a.bias ? *reinterpret_cast<const float4 *>(a.bias + n) : make_float4(0, 0, 0, 0);
            }
        const int next = tile + step;
        if (next < end) {
            aim(next / a.tiles_n * L::kM, next % a.tiles_n * L::kN);
            fetch(buffer ^ 1, 0);
        }
        multiply(buffer, left);
        workgroup_barrier();
        inside = m0 + L::kM <= M && n0 + L::kN <= N;
        // a lane's outputs: row r32 of X, columns 8 g + 4 half .. + 3 of W's 32.  They become rows in the wavefront's own part of
        // the buffer that is free now.
        constexpr int kRowPieces = TN * 4;
        _Float16 *out = reinterpret_cast<_Float16 *>(smem + buffer * L::kStage) + wave * (32 * L::kPitch);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float scale[4] = {sw[j][g].x, sw[j][g].y, sw[j][g].z, sw[j][g].w}, bias[4] = {b[j][g].x, b[j][g].y, b[j][g].z, b[j][g].w};
                    half4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = fmaf(static_cast<float>(acc[i][j][4 * g + e]), sx[i] * scale[e], bias[e]);
                        v = kGelu ? gelu(v) : v;
                        // (fp32 first: where the compiler makes one instruction of the last operation and the conversion, as it
                        // does for some tiles, a number in 70,000 is the other neighbour of a tie)
                        asm volatile("" : "+v"(v));
                        o[e] = static_cast<_Float16>(v);
                    }
                    *reinterpret_cast<half4 *>(out + r32 * L::kPitch + j * 32 + 8 * g + 4 * half) = o;
                }
            wave_fence();
#pragma unroll
            for (int t = 0; t < 2 * TN; ++t) {
                const int e = t * 64 + lane, r = e / kRowPieces, n = e % kRowPieces * 8;
                const half8 v = *reinterpret_cast<const half8 *>(out + r * L::kPitch + n);
                if (inside || (m0 + wave_m + i * 32 + r < M && n0 + wave_n + n < N))
                    *reinterpret_cast<half8 *>(a.y + static_cast<int64_t>(m0 + wave_m + i * 32 + r) * N + n0 + wave_n + n) = v;
            }
            wave_fence();
        }
        buffer ^= 1;
    }
}

template <typename L>
int launch(Int8Args a, bool gelu, hipStream_t stream)
{
    a.tiles_n = (a.N + L::kN - 1) / L::kN;
    const int64_t tiles = ceil_div(a.M, L::kM) * a.tiles_n;
    if (tiles > (1 << 30)) return fail(S3D_ERR_BAD_SHAPE, "s3d_linear_int8: M = %d rows", a.M);
    a.tiles = static_cast<int>(tiles);
    auto kernel = gelu ? linear_int8_kernel<L, true> : linear_int8_kernel<L, false>;
    // as many workgroups as fit the chip (by LDS), or one a tile
    constexpr int kPerCu = 160 * 1024 / L::kLds < 2 ? 1 : 160 * 1024 / L::kLds < 4 ? 160 * 1024 / L::kLds : 4;
    const int64_t slots = static_cast<int64_t>(kPerCu) * device_cus();
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(tiles < slots ? tiles : slots, 8) * 8)), dim3(kThreads), 0, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

}  // namespace

int launch_linear_int8(const LinearInt8 &l, hipStream_t stream)
{
    if (l.M < 0 || l.M > 0x7fffffff || l.N < 8 || l.N % 8 || l.K < 16 || l.K % 16 || l.K > 65536)
        return fail(S3D_ERR_BAD_SHAPE, "s3d_linear_int8: M=%lld N=%d K=%d (N a multiple of 8, K of 16 and at most 65536)", (long long)l.M, l.N, l.K);
    if (l.M == 0) return S3D_OK;
    if (!l.x || !l.sx || !l.w || !l.sw || !l.y) return fail(S3D_ERR_NULL_POINTER, "s3d_linear_int8: null device pointer");
    const Int8Args a{l.x, l.w, l.sx, l.sw, l.bias, static_cast<_Float16 *>(l.y), static_cast<int32_t>(l.M), l.N, l.K, 0, 0};
    const int64_t small = ceil_div(l.M, 64) * ((l.N + 63) / 64);
    if (small < (l.gelu ? 1024 : 576)) return launch<Tile<2, 2, 1, 1>>(a, l.gelu, stream);
    return launch<Tile<2, 2, 2, 1>>(a, l.gelu, stream);
}

namespace {

// The hidden layer in fp16, then its codes and scales
struct MlpPlaces {
    size_t hidden, codes, scales, total;
};

MlpPlaces places_of(int64_t M, int32_t hidden)
{
    MlpPlaces p{};
    const size_t numbers = static_cast<size_t>(M) * hidden;
    p.codes = p.hidden + align_up(2 * numbers, 256);
    p.scales = p.codes + align_up(numbers, 256);
    p.total = p.scales + align_up(static_cast<size_t>(M) * 4, 256);
    return p;
}

bool mlp_fits(int64_t M, int32_t C, int32_t hidden)
{
    return M >= 0 && M <= 0x7fffffff && C >= 16 && C % 16 == 0 && C <= 8192 && hidden >= 16 && hidden % 16 == 0 && hidden <= 8192;
}

}  // namespace
}  // namespace s3d

extern "C" __attribute__((visibility("default"))) int s3d_linear_int8(const int8_t *x, const float *x_scales, const int8_t *w, const float *w_scales,
                                                                      const float *bias, void *y, int64_t M, int32_t N, int32_t K, int32_t gelu,
                                                                      void *stream)
{
    return s3d::launch_linear_int8(s3d::LinearInt8{x, w, x_scales, w_scales, bias, y, M, N, K, gelu != 0}, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) size_t s3d_mlp_int8_workspace_bytes(int64_t M, int32_t C, int32_t hidden)
{
    return s3d::mlp_fits(M, C, hidden) ? s3d::places_of(M, hidden).total : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_mlp_int8(
    const int8_t *x, const float *x_scales, const int8_t *w1, const float *w1_scales, const float *b1, const int8_t *w2, const float *w2_scales,
    const float *b2, void *y, int64_t M, int32_t C, int32_t hidden, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace s3d;
    if (!mlp_fits(M, C, hidden))
        return fail(S3D_ERR_BAD_SHAPE, "s3d_mlp_int8: M=%lld C=%d hidden=%d (multiples of 16, at most 8192)", (long long)M, C, hidden);
    if (M == 0) return S3D_OK;
    const MlpPlaces p = places_of(M, hidden);
    if (!workspace || workspace_bytes < p.total)
        return fail(S3D_ERR_WORKSPACE, "s3d_mlp_int8: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), p.total);
    char *base = static_cast<char *>(workspace);
    int8_t *codes = reinterpret_cast<int8_t *>(base + p.codes);
    float *scales = reinterpret_cast<float *>(base + p.scales);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (int rc = launch_linear_int8({x, w1, x_scales, w1_scales, b1, base + p.hidden, M, hidden, C, true}, s)) return rc;
    if (int rc = launch_quantize_rows(base + p.hidden, S3D_DTYPE_F16, codes, scales, M, hidden, s)) return rc;
    return launch_linear_int8({codes, w2, scales, w2_scales, b2, y, M, C, hidden, false}, s);
}
