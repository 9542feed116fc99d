// Y = X W^T + b of rows in eight bits, with GELU on request (gfx950):
//   y[m][n] = sx[m] sw[n] (sum over k of x[m][k] w[n][k]) + b[n]
// x and w whole numbers -127 .. 127, the sum in 32 bits and exact, scales, bias and GELU in fp32, one rounding to fp16.
//
// The plan of linear.hip with bytes in place of fp16 numbers: a chunk is 128 numbers of K of a tile's rows of X and W, in LDS by direct
// loads, and a step of v_mfma_i32_32x32x32_i8 takes 32 of them, sixteen (a piece of 16 bytes) from each half of the lanes.  K is a
// multiple of 16: where half a step is left, the upper lanes put in zeros.
//
// Short sums are bound by the rows' memory (149,993 rows, 160 to 480, 42 us, 4.0 TB/s; 199,327, 48 to 192 with GELU, 26.8, 3.2, GELU's instructions beside
// it), long ones by LDS and the wait for a chunk (37,499, 1280 to 320, 26.2 us, 1.2 of 2.1 POP/s that a large product reaches), few rows by one tile's chunks
// one after the other (390, 640 to 1920, 5.1 us).
#include "attn_kernels.h"
#include "dense.h"
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
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
    // scales and biases of a tile's columns, in pieces of four: as many wavefronts fetch them
    static constexpr int kEnds = (kN / 2 + 63) / 64, kEndBytes = kEnds * 1024;
    static constexpr int kLds = 2 * kStage + 2 * kEndBytes;
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
    // what the end of a tile reads: the scales, then the biases of its columns, one tile ahead
    const int end_piece = wave * 64 + lane;
    auto fetch_ends = [&](int which, int n0) {
        if (wave >= L::kEnds) return;
        const int p = min(end_piece, L::kN / 2 - 1), q = p % (L::kN / 4);
        const float *at = p < L::kN / 4 || !a.bias ? a.sw : a.bias;
        load_to_lds(lds + 2 * L::kStage + which * L::kEndBytes + wave * 1024, at + min(n0 + 4 * q, N - 4));
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
    int ends = 0;
    aim(tile / a.tiles_n * L::kM, tile % a.tiles_n * L::kN);
    fetch_ends(0, tile % a.tiles_n * L::kN);
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
        // the rows' scales, before the next tile's first chunk: loads return in order
        float sx[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) sx[i] = a.sx[min(m0 + wave_m + i * 32 + r32, M - 1)];
        const int next = tile + step;
        if (next < end) {
            aim(next / a.tiles_n * L::kM, next % a.tiles_n * L::kN);
            fetch_ends(ends ^ 1, next % a.tiles_n * L::kN);
            fetch(buffer ^ 1, 0);
        }
        multiply(buffer, left);
        workgroup_barrier();
        inside = m0 + L::kM <= M && n0 + L::kN <= N;
        // a lane's outputs: row r32 of X, columns 8 g + 4 half .. + 3 of W's 32.  They become rows in the wavefront's own part of
        // the buffer that is free now.
        constexpr int kRowPieces = TN * 4;
        const f32x4 *sw = reinterpret_cast<const f32x4 *>(smem + 2 * L::kStage + ends * L::kEndBytes) + (wave_n + 4 * half) / 4, *biases = sw + L::kN / 4;
        _Float16 *out = reinterpret_cast<_Float16 *>(smem + buffer * L::kStage) + wave * (32 * L::kPitch);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 scale = sw[8 * j + 2 * g], bias = a.bias ? biases[8 * j + 2 * g] : f32x4{0, 0, 0, 0};
                    half4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = fmaf(static_cast<float>(acc[i][j][4 * g + e]), sx[i] * scale[e], bias[e]);
                        o[e] = to_half(kGelu ? gelu(v) : v);
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
        ends ^= 1;
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

// A tile of 32 x 32 whose chunks are shared by eight wavefronts, wavefront s taking chunks s, s + 8, .. through an LDS buffer of its
// own (no barrier), two chunks ahead in registers; the sums meet in LDS.  For launches whose larger tiles would leave CUs without work.
constexpr int kShares = 8;

template <bool kGelu>
__global__ __launch_bounds__(64 * kShares) void linear_int8_thin_kernel(Int8Args a)
{
    constexpr int kOwn = 2 * 32 * kChunk, kPitch = 32 + 4;
    static_assert(32 * kPitch * 4 <= kOwn, "a wavefront's sums fit its buffer");
    __shared__ __align__(16) char smem[kShares * kOwn];
    const int M = a.M, N = a.N, K = a.K;
    // workgroups b, b + 8, .. run on one XCD: they get neighbouring tiles, which share rows of X
    const int share = (a.tiles + 7) / 8, tile = static_cast<int>(blockIdx.x) % 8 * share + static_cast<int>(blockIdx.x) / 8;
    if (tile >= a.tiles) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, half = lane >> 5;
    const int m0 = tile / a.tiles_n * 32, n0 = tile % a.tiles_n * 32, chunks = (K + kChunk - 1) / kChunk;
    char *own = smem + wave * kOwn;

    const int piece = lane % kPieces, row = lane / kPieces;      // rows row + 8 i: of X, then of W
    const int8_t *from[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = row + 8 * (i % 4);
        from[i] = (i < 4 ? a.x + static_cast<int64_t>(min(m0 + r, M - 1)) * K : a.w + static_cast<int64_t>(min(n0 + r, N - 1)) * K) + piece * 16;
    }
    i32x16 acc = {};
    // (pieces behind K are zeros)
    auto fetch = [&](uint4 (&held)[8], int chunk) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            held[i] = chunk * kChunk + piece * 16 < K ? *reinterpret_cast<const uint4 *>(from[i] + chunk * kChunk) : make_uint4(0, 0, 0, 0);
    };
    auto multiply = [&](uint4 (&held)[8], int chunk) {
        uint4 *to = reinterpret_cast<uint4 *>(own);
#pragma unroll
        for (int i = 0; i < 8; ++i) to[placed(row + 8 * i, piece)] = held[i];
        fetch(held, chunk + 2 * kShares);
        wave_fence();
        const i32x4 *at = reinterpret_cast<const i32x4 *>(own);
        const int left = K - chunk * kChunk;
#pragma unroll
        for (int s = 0; s < kChunk / 32; ++s) {
            if (32 * s >= left) break;
            acc = product(at[placed(32 + r32, 2 * s + half)], at[placed(r32, 2 * s + half)], acc);
        }
        wave_fence();
    };
    uint4 first[8], second[8];
    fetch(first, wave);
    fetch(second, wave + kShares);
    const int n = n0 + threadIdx.x % 16 * 2, r = threadIdx.x / 16;
    const int end = min(n, N - 2);
    const float2 sw = *reinterpret_cast<const float2 *>(a.sw + end), bias = a.bias ? *reinterpret_cast<const float2 *>(a.bias + end) : make_float2(0, 0);
    const float sx = a.sx[min(m0 + r, M - 1)];
    for (int chunk = wave; chunk < chunks; chunk += 2 * kShares) {
        multiply(first, chunk);
        if (chunk + kShares < chunks) multiply(second, chunk + kShares);
    }
    int *sums = reinterpret_cast<int *>(own);
#pragma unroll
    for (int g = 0; g < 4; ++g)
        *reinterpret_cast<int4 *>(sums + r32 * kPitch + 8 * g + 4 * half) = make_int4(acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]);
    __syncthreads();
    static_assert(4 * kShares == 32, "a row for sixteen threads");
    int v[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kShares; ++i) {
        const int2 part = *reinterpret_cast<const int2 *>(smem + i * kOwn + (r * kPitch + threadIdx.x % 16 * 2) * 4);
        v[0] += part.x;
        v[1] += part.y;
    }
    half2 o;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float z = fmaf(static_cast<float>(v[e]), sx * (e ? sw.y : sw.x), e ? bias.y : bias.x);
        o[e] = to_half(kGelu ? gelu(z) : z);
    }
    if (m0 + r < M && n < N) *reinterpret_cast<half2 *>(a.y + static_cast<int64_t>(m0 + r) * N + n) = o;
}

int launch_thin(Int8Args a, bool gelu, hipStream_t stream)
{
    a.tiles_n = (a.N + 31) / 32;
    const int64_t tiles = ceil_div(a.M, 32) * a.tiles_n;
    a.tiles = static_cast<int>(tiles);
    auto kernel = gelu ? linear_int8_thin_kernel<true> : linear_int8_thin_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(tiles, 8) * 8)), dim3(64 * kShares), 0, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

// Weights in LDS, rows in registers.  A workgroup fetches the weights once.  After that its eight wavefronts
// take 32 rows at a time, as many wavefronts of the same rows as share out the columns; the rows' pieces come from memory in the lanes
// that the products want them in, those of the next step meanwhile.  The results of a step meet in LDS and leave as one run of whole
// rows: lines of 128 bytes that are written in parts, as those at the ends of a row's 64 or 128 columns are where N is no multiple of 64,
// cost as much as half as many lines more (595,677 rows, 80 to 256 channels, 81 us, to 240 118, a wavefront's 64 columns at a time).
constexpr int kRowsThreads = 512, kRowsWaves = kRowsThreads / 64, kRowsLds = 160 * 1024, kRowsStage = 52 * 1024;

struct Int8Slices {
    int columns, groups;      // a multiple of 64, N at least; workgroups
    int sharing;              // wavefronts of the same rows
};

template <int STEPS> constexpr int rows_pitch() { return (2 * STEPS) | 1; }      // pieces of a row of weights: sixteen rows' lie in all banks
__host__ __device__ constexpr int rows_stage_pitch(int columns) { return columns + 8; }
inline int rows_stage(int columns, int sharing) { return kRowsWaves / sharing * 32 * rows_stage_pitch(columns) * 2; }
template <int STEPS> int rows_lds(const Int8Slices &s) { return s.columns * (rows_pitch<STEPS>() * 16 + 8) + rows_stage(s.columns, s.sharing); }

template <int STEPS, bool kGelu>
__global__ __launch_bounds__(kRowsThreads, 4) void linear_int8_rows_kernel(Int8Args a, Int8Slices slices)
{
    extern __shared__ __align__(16) char dynamic[];
    constexpr int kPitch = rows_pitch<STEPS>();
    i32x4 *weights = reinterpret_cast<i32x4 *>(dynamic);
    float *scales = reinterpret_cast<float *>(weights + slices.columns * kPitch), *biases = scales + slices.columns;
    _Float16 *stage = reinterpret_cast<_Float16 *>(biases + slices.columns);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, half = lane >> 5;
    const int M = a.M, N = a.N, K = a.K;
    const int sub = wave / slices.sharing, first_tile = wave % slices.sharing, rows_a_step = kRowsWaves / slices.sharing * 32;
    const int steps = (M - 1) / rows_a_step + 1;      // (M up to 2^31 - 1)
    int at_step = static_cast<int>(blockIdx.x);
    if (at_step >= steps) return;

    i32x4 rows[STEPS], next[STEPS];
    float sx, next_sx;
    auto fetch = [&](i32x4 (&to)[STEPS], float &scale, int which) {
        const int m = min(which * rows_a_step + sub * 32 + r32, M - 1);
        const int8_t *from = a.x + static_cast<int64_t>(m) * K;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int k = 32 * s + 16 * half;
            to[s] = *reinterpret_cast<const i32x4 *>(from + (k < K ? k : 0));      // (beyond K the weights are zeros)
        }
        scale = a.sx[m];
    };
    fetch(rows, sx, at_step);
    for (int i = tid; i < slices.columns * 2 * STEPS; i += kRowsThreads) {
        const int n = i / (2 * STEPS), p = i % (2 * STEPS);
        i32x4 v = {0, 0, 0, 0};
        if (n < N && 16 * p < K) v = *reinterpret_cast<const i32x4 *>(a.w + static_cast<int64_t>(n) * K + 16 * p);
        weights[n * kPitch + p] = v;
    }
    for (int n = tid; n < slices.columns; n += kRowsThreads) {
        scales[n] = n < N ? a.sw[n] : 0.0f;
        biases[n] = n < N && a.bias ? a.bias[n] : 0.0f;
    }
    const int pitch = rows_stage_pitch(slices.columns), pieces = N / 8;
    const uint32_t magic = ((1u << 20) + pieces - 1) / pieces;      // p / pieces = p magic / 2^20 for p pieces < 2^20
    _Float16 *own = stage + (sub * 32 + r32) * pitch + 4 * half;
    __syncthreads();
    for (; at_step < steps; at_step += slices.groups) {
        fetch(next, next_sx, min(at_step + slices.groups, steps - 1));
        for (int c = first_tile * 32; c < N; c += slices.sharing * 32) {
            i32x16 acc = {};
            const i32x4 *at = weights + (c + r32) * kPitch + half;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) acc = product(at[2 * s], rows[s], acc);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = c + 8 * g + 4 * half;
                const f32x4 scale = *reinterpret_cast<const f32x4 *>(scales + n), bias = *reinterpret_cast<const f32x4 *>(biases + n);
                half4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = fmaf(static_cast<float>(acc[4 * g + e]), sx * scale[e], bias[e]);
                    o[e] = to_half(kGelu ? gelu(v) : v);
                }
                *reinterpret_cast<half4 *>(own + c + 8 * g) = o;
            }
        }
        // The next rows are there before these are stored: a wait for them behind the stores would be one for the stores too.
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            asm volatile("" : "+v"(next[s]));
            rows[s] = next[s];
        }
        asm volatile("" : "+v"(next_sx));
        sx = next_sx;
        workgroup_barrier();
        const int m0 = at_step * rows_a_step, count = min(rows_a_step, M - m0) * pieces;
        _Float16 *to = a.y + static_cast<int64_t>(m0) * N;
        for (int p = tid; p < count; p += kRowsThreads) {
            const int r = static_cast<int>(p * magic >> 20), n = (p - r * pieces) * 8;
            *reinterpret_cast<half8 *>(to + r * N + n) = *reinterpret_cast<const half8 *>(stage + r * pitch + n);
        }
        workgroup_barrier();
    }
}

// One slice, as few wavefronts of the same rows as their results leave room for, or more where that lets two workgroups on a CU (us,
// 100,000 rows of 96 to 384 with GELU 32.3 / 27.1)
template <int STEPS> Int8Slices rows_slices(int N)
{
    Int8Slices s{(N + 63) / 64 * 64, 0, 1};
    while (s.sharing < kRowsWaves && rows_stage(s.columns, s.sharing) > kRowsStage) s.sharing *= 2;
    for (Int8Slices more = s; more.sharing < kRowsWaves;) {
        more.sharing *= 2;
        if (2 * rows_lds<STEPS>(s) > kRowsLds && 2 * rows_lds<STEPS>(more) <= kRowsLds) return more;
    }
    return s;
}

template <int STEPS> int launch_rows_of(Int8Args a, bool gelu, hipStream_t stream)
{
    Int8Slices slices = rows_slices<STEPS>(a.N);
    const int lds = rows_lds<STEPS>(slices), per_cu = 2 * lds <= kRowsLds ? 2 : 1;
    const int64_t steps = ceil_div(a.M, kRowsWaves / slices.sharing * 32), most = static_cast<int64_t>(per_cu) * device_cus();
    slices.groups = static_cast<int>(ceil_div(steps < most ? steps : most, 8) * 8);
    auto kernel = gelu ? linear_int8_rows_kernel<STEPS, true> : linear_int8_rows_kernel<STEPS, false>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), kRowsLds)) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(slices.groups)), dim3(kRowsThreads), lds, stream, a, slices);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

// Where the weights fit LDS and a workgroup has rows enough for what it takes to fetch them.  us, tiles / so: 595,677 rows, 80 to 240
// 99 / 69, to 320 with GELU 146 / 127; 199,327, 48 to 144 18.4 / 14.3, to 192 with GELU 30.4 / 29.3; 149,993, 160 to 480 56.7 / 44.5, to
// 640 with GELU 83 / 75, to 160 18.7 / 18.2; 49,682, 96 to 288 10.6 / 10.4; below N K rows 1.0 to 1.4 times as long (50,000, 192 to 576,
// 19.6 / 23.8), beyond 192 channels 0.95 to 1.7 times.
bool rows_pay(const Int8Args &a)
{
    if (a.K > 192 || a.M < 32768 || a.M < static_cast<int64_t>(a.N) * a.K) return false;
    switch ((a.K + 31) / 32) {
#define S3D_CASE(S) case S: return rows_lds<S>(rows_slices<S>(a.N)) <= kRowsLds;
        S3D_CASE(1) S3D_CASE(2) S3D_CASE(3) S3D_CASE(4) S3D_CASE(5) S3D_CASE(6)
#undef S3D_CASE
    }
    return false;
}

int launch_rows(const Int8Args &a, bool gelu, hipStream_t stream)
{
    switch ((a.K + 31) / 32) {
#define S3D_CASE(S) case S: return launch_rows_of<S>(a, gelu, stream);
        S3D_CASE(1) S3D_CASE(2) S3D_CASE(3) S3D_CASE(4) S3D_CASE(5) S3D_CASE(6)
#undef S3D_CASE
    }
    return fail(S3D_ERR_BAD_SHAPE, "s3d_linear_int8: K=%d", a.K);
}

}  // namespace

int launch_linear_int8(const LinearInt8 &l, hipStream_t stream)
{
    if (l.M < 0 || l.M > 0x7fffffff || l.N < 8 || l.N % 8 || l.K < 16 || l.K % 16 || l.K > 65536)
        return fail(S3D_ERR_BAD_SHAPE, "s3d_linear_int8: M=%lld N=%d K=%d (N a multiple of 8, K of 16 and at most 65536)", (long long)l.M, l.N, l.K);
    if (l.M == 0) return S3D_OK;
    if (!l.x || !l.sx || !l.w || !l.sw || !l.y) return fail(S3D_ERR_NULL_POINTER, "s3d_linear_int8: null device pointer");
    const Int8Args a{l.x, l.w, l.sx, l.sw, l.bias, static_cast<_Float16 *>(l.y), static_cast<int32_t>(l.M), l.N, l.K, 0, 0};
    // Tiles of 32 x 32 with K shared as long as each has a CU, or half of one with long sums.  us, 64 x 64 / so: 1 row, 2560 to 640, 7.4 / 4.5;
    // 100, 1536 to 384 5.7 / 4.0, 384 to 384 4.1 / 3.8; 390, 2560 to 640 (260 tiles) 7.7 / 6.8, 384 to 384 4.1 / 4.0; 1,563, 1280 to 320
    // (490) 5.5 / 5.4; 811, 640 to 640 (520) 5.9 / 5.8, 384 to 1152 (936) 4.0 / 6.1, 2560 to 640 8.0 / 9.0.
    const int64_t thin = ceil_div(l.M, 32) * ((l.N + 31) / 32);
    if (thin <= 256 || (thin <= 512 && l.K >= 1024)) return launch_thin(a, l.gelu, stream);
    if (rows_pay(a)) return launch_rows(a, l.gelu, stream);
    // Tiles of 64 x 64 as long as larger ones would leave CUs without work (us, 64 x 64 / 128 x 64, by their number: 585 5.1 / 5.6, 980
    // 7.4 / 8.3, 882 6.4 / 5.9, 1440 12.5 / 11.6, 1470 8.6 / 7.9, 1565 19.2 / 19.4, 3130 26.5 / 20.2); then 128 rows by 128 columns where that pads
    // N no more than 64 (128 x 64 / so: 20,000 rows, 640 to 1920 50.9 / 46.2; 100,000, 256 to 384 36.1 / 32.7; 60,000, 192 to 768 with GELU
    // 45.2 / 43.0; 37,499, 320 to 1280 with GELU 53.7 / 52.8), by 96 likewise (60,000, 192 to 576 24.8 / 22.5; 100,000, 384 to 96 16.2 / 13.6;
    // 6,250, 320 to 960 7.9 / 7.5), else by 64.  With GELU, whose instructions more wavefronts hide, up to 320 channels 64 x 64 up to 6144 of them
    // (12,421, 192 to 768 11.7 / 11.1; 49,682, 96 to 384 17.3 / 16.6), and never 96 (18.9, 13.2).
    const int64_t small = ceil_div(l.M, 64) * ((l.N + 63) / 64);
    if (small < 1024 || (l.gelu && l.K <= 320 && small <= 6144)) return launch<Tile<2, 2, 1, 1>>(a, l.gelu, stream);
    auto padded = [&](int width) { return (l.N + width - 1) / width * width; };
    if (padded(128) == padded(64) && ceil_div(l.M, 128) * (padded(128) / 128) >= 640) return launch<Tile<2, 2, 2, 2>>(a, l.gelu, stream);
    if (padded(96) <= padded(64) && !l.gelu) return launch<Tile<4, 1, 1, 3>>(a, l.gelu, stream);
    return launch<Tile<4, 1, 1, 2>>(a, l.gelu, stream);
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
    return s3d::mlp_fits(M, C, hidden) && !s3d::mlp_int8_pays(M, C, hidden) ? s3d::places_of(M, hidden).total : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_mlp_int8(
    const int8_t *x, const float *x_scales, const int8_t *w1, const float *w1_scales, const float *b1, const int8_t *w2, const float *w2_scales,
    const float *b2, void *y, int64_t M, int32_t C, int32_t hidden, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace s3d;
    if (!mlp_fits(M, C, hidden))
        return fail(S3D_ERR_BAD_SHAPE, "s3d_mlp_int8: M=%lld C=%d hidden=%d (multiples of 16, at most 8192)", (long long)M, C, hidden);
    if (M == 0) return S3D_OK;
    if (mlp_int8_pays(M, C, hidden)) {
        if (!x || !x_scales || !w1 || !w1_scales || !w2 || !w2_scales || !y) return fail(S3D_ERR_NULL_POINTER, "s3d_mlp_int8: null device pointer");
        return launch_mlp_int8({x, w1, w2, x_scales, w1_scales, b1, w2_scales, b2, y, M, C, hidden}, static_cast<hipStream_t>(stream));
    }
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
