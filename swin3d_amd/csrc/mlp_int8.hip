// Both layers of an MLP of rows in eight bits as one kernel (gfx950):
//   h = GELU(sx s1 (x w1^T) + b1) rounded to fp16, in eight bits by its row's largest number, y = sh s2 (h w2^T) + b2
// with the operations, and so the bits, of linear_int8.hip's layers and norm_int8.hip's rows one after the other.
//
// A row's codes need its largest number, so a workgroup has whole rows of the hidden layer, 32 or 64, whose columns its wavefronts
// share in tiles of 32.  They stay in registers as fp16 numbers, two a register, until the wavefronts have met with the rows' largest,
// and are written once, as codes, to LDS, from where the second product reads them.  In memory are x, y and the weights alone; those
// come from L2 for every workgroup, through a buffer of a wavefront's own, a chunk ahead.
// Few rows are bound by what a wavefront waits for its weights, many by GELU and the codes, thirty instructions a number.  12,421 rows of 192 over 768
// 18.8 us, 0.39 POP/s; 595,677 of 80 over 320 233.
#include "attn_kernels.h"
#include "dense.h"
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kChunk = 16 * kPieces, kStage = 32 * kChunk;      // numbers of K staged at a time, bytes of a tile's chunk
constexpr int kLds = 160 * 1024;

constexpr int up_to(int n, int step) { return (n + step - 1) / step * step; }

struct Places {
    int x_pitch, h_pitch, h, ends, most, total;      // bytes: of a row of x and of the hidden layer, odd numbers of pieces; where things are
};
__host__ __device__ inline Places places_of(int C, int hidden, int waves, int rows)
{
    Places p{};
    const int c = up_to(C, 32), n = up_to(hidden, 32);
    p.x_pitch = c + 16;
    p.h_pitch = n + 16;
    int at = 2 * waves * kStage + rows * p.x_pitch;
    p.h = at;
    const int codes = rows * p.h_pitch, results = rows * (2 * C + 16);      // (the results take the codes' place)
    at += codes > results ? codes : results;
    p.ends = at;      // scales and biases of both layers, zeros behind the last column
    at += 2 * (n + c) * 4;
    p.most = at;
    p.total = at + waves * rows * 4;
    return p;
}

constexpr int kTiles2 = 2;      // of the second product a wavefront

template <int WAVES, int R, int TILES>
__global__ __launch_bounds__(64 * WAVES, 2) void mlp_int8_kernel(MlpInt8 a)
{
    extern __shared__ __align__(16) char smem[];
    constexpr int kThreads = 64 * WAVES, kWaves = WAVES, kRows = 32 * R;
    const int C = a.C, hidden = a.hidden, M = static_cast<int>(a.M);
    const Places p = places_of(C, hidden, WAVES, kRows);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, half = lane >> 5;
    const int m0 = static_cast<int>(blockIdx.x) * kRows;
    char *rows = smem + 2 * kWaves * kStage, *own = smem + wave * (2 * kStage);
    float *scales1 = reinterpret_cast<float *>(smem + p.ends), *biases1 = scales1 + up_to(hidden, 32), *scales2 = biases1 + up_to(hidden, 32),
          *biases2 = scales2 + up_to(C, 32);
    uint32_t *most_of = reinterpret_cast<uint32_t *>(smem + p.most);
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem)) + wave * (2 * kStage);

    // Chunk k0 of the 32 rows from n0 on of a weight [N,K]: an instruction takes eight rows.  A piece behind K is the chunk's first one,
    // which meets zeros.
    auto fetch = [&](int buffer, const int8_t *w, int N, int K, int n0, int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = lane / kPieces + 8 * i, piece = (lane ^ (r >> 1)) & (kPieces - 1);
            const uint32_t at = static_cast<uint32_t>(min(n0 + r, N - 1) * K + k0 + (k0 + 16 * piece < K ? 16 * piece : 0));
            load_to_lds_from(lds + buffer * kStage + i * 1024, w, at);
        }
    };
    // The rows, of `pitch` bytes, times a tile of weights, of which the first chunk is under way; `then` sets out for what comes next
    int buffer = 0;
    auto tile_product = [&](i32x16 (&acc)[R], const char *from, int pitch, const int8_t *w, int N, int K, int n0, auto then) {
#pragma unroll
        for (int i = 0; i < R; ++i) acc[i] = i32x16{};
        const char *row = from + r32 * pitch + 16 * half;
        for (int k0 = 0; k0 < K; k0 += kChunk) {
            bool more = true;
            if (k0 + kChunk < K) fetch(buffer ^ 1, w, N, K, n0, k0 + kChunk);
            else more = then(buffer ^ 1);
            if (more) loads_done<4>();
            else loads_done<0>();
            const i32x4 *at = reinterpret_cast<const i32x4 *>(own + buffer * kStage);
#pragma unroll
            for (int s = 0; s < kChunk / 32; ++s) {
                if (k0 + 32 * s >= K) break;
                const i32x4 weights = at[placed(r32, 2 * s + half)];
#pragma unroll
                for (int i = 0; i < R; ++i)
                    acc[i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(weights, *reinterpret_cast<const i32x4 *>(row + 32 * i * pitch + k0 + 32 * s), acc[i], 0, 0, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // read before the next chunk but one is set out for
            buffer ^= 1;
        }
    };
    const int tiles1 = (hidden + 31) / 32, tiles2 = (C + 31) / 32;
    if (wave < tiles1) fetch(0, a.w1, hidden, C, 32 * wave, 0);

    const int pieces = up_to(C, 32) / 16;
    for (int i = tid; i < kRows * pieces; i += kThreads) {
        const int r = i / pieces, k = i % pieces * 16;
        i32x4 v = {0, 0, 0, 0};
        if (k < C) v = *reinterpret_cast<const i32x4 *>(a.x + static_cast<int64_t>(min(m0 + r, M - 1)) * C + k);
        *reinterpret_cast<i32x4 *>(rows + r * p.x_pitch + k) = v;
    }
    for (int n = tid; n < up_to(hidden, 32); n += kThreads) {
        scales1[n] = n < hidden ? a.s1[n] : 0.0f;
        biases1[n] = n < hidden && a.b1 ? a.b1[n] : 0.0f;
    }
    for (int n = tid; n < up_to(C, 32); n += kThreads) {
        scales2[n] = n < C ? a.s2[n] : 0.0f;
        biases2[n] = n < C && a.b2 ? a.b2[n] : 0.0f;
    }
    float sx[R];
#pragma unroll
    for (int i = 0; i < R; ++i) sx[i] = a.sx[min(m0 + 32 * i + r32, M - 1)];
    __syncthreads();

    // The hidden layer.  A lane has rows r32 + 32 i, columns 8 g + 4 half .. + 3 of a tile's 32.
    half4 u[TILES][R][4];
    uint32_t most[R] = {};
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int tile = wave + t * kWaves;
        if (tile >= tiles1) break;
        i32x16 acc[R];
        tile_product(acc, rows, p.x_pitch, a.w1, hidden, C, 32 * tile, [&](int into) {
            if (tile + kWaves < tiles1) fetch(into, a.w1, hidden, C, 32 * (tile + kWaves), 0);
            else if (wave < tiles2) fetch(into, a.w2, C, hidden, 32 * wave, 0);
            else return false;
            return true;
        });
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = 32 * tile + 8 * g + 4 * half;
            const f32x4 scale = *reinterpret_cast<const f32x4 *>(scales1 + n), bias = *reinterpret_cast<const f32x4 *>(biases1 + n);
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) u[t][i][g][e] = to_half(gelu(fmaf(static_cast<float>(acc[i][4 * g + e]), sx[i] * scale[e], bias[e])));
                const uint2 w = __builtin_bit_cast(uint2, u[t][i][g]);
                const uint32_t pair = larger_pair(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
                most[i] = max(most[i], max(pair >> 16, pair & 0xffffu));
            }
        }
    }
    // (a wavefront without a tile of the hidden layer may have one of the second product)
    if (wave >= tiles1 && wave < tiles2) fetch(0, a.w2, C, hidden, 32 * wave, 0);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const auto swapped = __builtin_amdgcn_permlane32_swap(most[i], most[i], false, false);
        if (half == 0) most_of[wave * kRows + 32 * i + r32] = max(swapped[0], swapped[1]);
    }
    workgroup_barrier();
    char *codes = smem + p.h;
    float sh[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        uint32_t largest = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) largest = max(largest, most_of[w * kRows + 32 * i + r32]);
        const bool finite = largest < 0x7c00u;
        const float a_max = finite ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(largest))) : 0.0f;
        const float reciprocal = a_max > 0.0f ? 1.0f / a_max : 0.0f, inverse = a_max > 0.0f ? 127.0f / a_max : 0.0f;
        sh[i] = finite ? a_max / 127.0f : __builtin_nanf("");
        // 127 u / a_max correctly rounded, so that ties, which rows of fp16 numbers have, go to even
        auto code = [&](float number) {
            const float q = number * inverse;
            return __float_as_uint(finite ? fmaf(fmaf(-q, a_max, 127.0f * number), reciprocal, q) + 12582912.0f : 0.0f);
        };
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int tile = wave + t * kWaves;
            if (tile >= tiles1) break;
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint32_t *>(codes + (32 * i + r32) * p.h_pitch + 32 * tile + 8 * g + 4 * half) =
                    four_bytes(code(u[t][i][g][0]), code(u[t][i][g][1]), code(u[t][i][g][2]), code(u[t][i][g][3]));
        }
    }
    workgroup_barrier();

    // The second product.  Its results wait in registers until nobody reads codes any more.
    half4 o[kTiles2][R][4];
#pragma unroll
    for (int t = 0; t < kTiles2; ++t) {
        const int tile = wave + t * kWaves;
        if (tile >= tiles2) break;
        i32x16 acc[R];
        tile_product(acc, codes, p.h_pitch, a.w2, C, hidden, 32 * tile, [&](int into) {
            if (tile + kWaves >= tiles2) return false;
            fetch(into, a.w2, C, hidden, 32 * (tile + kWaves), 0);
            return true;
        });
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = 32 * tile + 8 * g + 4 * half;
            const f32x4 scale = *reinterpret_cast<const f32x4 *>(scales2 + n), bias = *reinterpret_cast<const f32x4 *>(biases2 + n);
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][i][g][e] = to_half(fmaf(static_cast<float>(acc[i][4 * g + e]), sh[i] * scale[e], bias[e]));
        }
    }
    workgroup_barrier();
    const int pitch = C + 8;
    _Float16 *results = reinterpret_cast<_Float16 *>(codes);
#pragma unroll
    for (int t = 0; t < kTiles2; ++t) {
        const int tile = wave + t * kWaves;
        if (tile >= tiles2) break;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = 32 * tile + 8 * g + 4 * half;
            if (n >= C) continue;
#pragma unroll
            for (int i = 0; i < R; ++i) *reinterpret_cast<half4 *>(results + (32 * i + r32) * pitch + n) = o[t][i][g];
        }
    }
    workgroup_barrier();
    const int eights = C / 8, count = min(kRows, M - m0) * eights;
    _Float16 *to = static_cast<_Float16 *>(a.y) + static_cast<int64_t>(m0) * C;
    for (int i = tid; i < count; i += kThreads) {
        const int r = i / eights, n = i % eights * 8;
        *reinterpret_cast<half8 *>(to + r * C + n) = *reinterpret_cast<const half8 *>(results + r * pitch + n);
    }
}

template <int WAVES, int R, int TILES> int launch_tiles(const MlpInt8 &a, hipStream_t stream)
{
    auto kernel = mlp_int8_kernel<WAVES, R, TILES>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), kLds)) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(a.M, 32 * R))), dim3(64 * WAVES), places_of(a.C, a.hidden, WAVES, 32 * R).total, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

constexpr int kMostTiles = 5;      // of the hidden layer a wavefront: more of them fit no LDS

template <int WAVES, int R> int launch_form(const MlpInt8 &a, hipStream_t stream)
{
    switch ((a.hidden + 32 * WAVES - 1) / (32 * WAVES)) {
#define S3D_CASE(T) case T: return launch_tiles<WAVES, R, T>(a, stream);
        S3D_CASE(1) S3D_CASE(2) S3D_CASE(3) S3D_CASE(4) S3D_CASE(5)
#undef S3D_CASE
    }
    return fail(S3D_ERR_BAD_SHAPE, "s3d_mlp_int8: %d hidden channels", a.hidden);
}

bool fits(int C, int hidden, int waves, int r, int lds)
{
    return hidden <= 32 * waves * kMostTiles && C <= 32 * waves * kTiles2 && places_of(C, hidden, waves, 32 * r).total <= lds;
}

}  // namespace

// Where LDS has room for 64 rows and eight wavefronts, but for few rows of wide layers, whose weights few workgroups fetch.  us, the layers apart / so,
// hidden = 4 C: 40 rows of 48 12.0 / 5.9, of 192 11.3 / 11.7, of 256 11.4 / 14.6; 1,600 of 256 14.9 / 15.4; 12,421 of 192 31.0 / 19.4; 49,682 of
// 256 99.6 / 95.9; 150,000 of 48 60.8 / 46.7, of 128 129 / 88, of 256 312 / 232; 595,677 of 80 353 / 233; 49,682, 320 to 640 77.5 / 79.1.
bool mlp_int8_pays(int64_t M, int32_t C, int32_t hidden) { return fits(C, hidden, 8, 2, kLds) && (M >= 1600 || C * hidden <= 160000); }

// 32 rows and eight wavefronts as long as each has a CU (us, eight / four wavefronts: 6,250 rows of 192 13.1 / 18.7, of 48 6.5 / 7.1; 64 rows 19.0), then 64,
// for which the weights come once: of four wavefronts where a CU has room for two such, or else of eight (25,000 rows of 128, 32 rows and four
// wavefronts 25.9, 64 and four 22.0, 64 and eight 25.9; 150,000 of 192 to 384 110, 85.2, 108, to 768 182, 246, 177; 12,421 of 160 19.4, 22.2, 16.2; most that
// 32 and four would give: 49,682 of 48 18.2, 20.7, 28.4, 150,000 of 96 to 768 139, 191, 158).
int launch_mlp_int8(const MlpInt8 &a, hipStream_t stream)
{
    const int64_t cus = device_cus();
    if (a.M <= 32 * cus) return launch_form<8, 1>(a, stream);
    if (a.M > 64 * cus && fits(a.C, a.hidden, 4, 2, kLds / 2)) return launch_form<4, 2>(a, stream);
    return launch_form<8, 2>(a, stream);
}

}  // namespace s3d
