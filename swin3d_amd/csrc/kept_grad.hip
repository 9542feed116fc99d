// Weight and bias gradients of layers that keep their input in eight bits (gfx950): dW = dY^T X', db = the column sums of dY, dY in fp16, X'
// what is kept (rows8.h) or rows in fp16, sums in fp32.
//
// The sum runs over the rows, but rows are what lies one behind the other: the matrix instruction wants eight rows' numbers of one
// column in a lane.  LDS gives them so (ds_read_b64_tr_b16: four rows' numbers of a column from four rows of four neighbouring numbers), and
// dY's pieces of 16 bytes go to LDS without a register between; X's codes become fp16 numbers on their way there, once for a workgroup's
// 128 columns of dY.  A block of 32 rows by 16 columns is 1024 bytes, its pieces (row r, half h) at place q(r, h) such that the pieces of one
// transposing read, two halves of eight rows four apart, lie in all banks.
//
// A workgroup has 128 or 64 columns of dY by 32 B of X and a share of the rows; its eight wavefronts have 32 columns of dY each, all of X's, and
// every second or fourth block of 32 rows.  The shares' parts are added by linear_grad.hip's second kernel: no atomics, the same bits on every call.
//
// Bound by memory where the widths are small (199,327 rows of 144 and 48 channels 19.5 us, 3.5 TB/s; 149,993 of 640 and 160 96 us kept, 85 in fp16, 2.3
// and 2.8 TB/s, with dY read for every 96 of X's columns in the first), by launch and sums where rows are few (811 of 1152 and 384 10.9 us).
#include "attn_kernels.h"
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __fp16 lds_half4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512, kWaves = kThreads / 64, kBlock = 1024;      // threads; bytes of a block

// One operand's columns are the tile's rows, those of the other its columns; turned, these are X's and dY's, and the tile is stored so.
struct GradArgs {
    const _Float16 *n;        // [M,N] fp16
    const void *k;            // [M,K] fp16, or kept
    float *parts;             // [splits][N K + N], turned [splits][N K + K]
    const float *sums;        // [ceil(M / 32)][N] or null: what the columns of dY add up to over each 32 rows (not turned)
    int64_t M, rows;          // rows of a split, a multiple of a stage's
    int N, K, tiles_k, tiles, splits;
    bool turned;
};

// of the finished sums, in numbers
constexpr int pitch_of(int b) { return 32 * b + 4; }

// An operand of a stage in LDS: blocks of kTall rows by kWide columns
template <int ROWS, int COLUMNS> struct Operand {
    static constexpr int kWide = COLUMNS % 64 == 0 ? 64 : 32, kTall = kBlock / 2 / kWide, kAcross = COLUMNS / kWide, kBlocks = ROWS / kTall * kAcross;
    // The place of piece p (eight columns) of row r of a block, and what is at a place.  The pieces of a row come from memory in one run: in any
    // other order the address unit takes up to twice as long for the stage (37,499 rows, 320 and 1280 columns, 52 us / 101).
    static constexpr int kRowPieces = kWide / 8;
    static __device__ __forceinline__ int turn(int r) { return kWide == 64 ? (r >> 1 & 1) << 2 : 0; }
    static __device__ __forceinline__ int place(int r, int p) { return r * kRowPieces + (p ^ turn(r)); }
    static __device__ __forceinline__ int row_at(int q) { return q / kRowPieces; }
    static __device__ __forceinline__ int piece_at(int q) { return q % kRowPieces ^ turn(q / kRowPieces); }
    // Where a lane asks for eight rows' numbers of a column, by two reads kNext apart: rows 8 half + 4 i .. + 3 by read i; sixteen lanes a block of
    // sixteen columns, lane l of them for row l / 4 and numbers 4 (l % 4) .. + 3; of 32 columns from 32 c on
    static constexpr int kNext = 4 * kRowPieces * 16;
    static __device__ __forceinline__ int asked(int lane, int c)
    {
        const int l = lane & 15, pieces = (kWide == 64 ? c % 2 * 4 : 0) + 2 * (lane >> 4 & 1) + (l >> 1 & 1);
        return place(l >> 2, pieces) * 16 + (l & 1) * 8 + (lane >> 5) * (kWide == 64 ? kAcross * kBlock : 512);
    }
    // ... and of the sixteen rows from 16 s on
    static __device__ __forceinline__ int start(int s, int c) { return kWide == 64 ? (2 * s * kAcross + c / 2) * kBlock : (s * kAcross + c) * kBlock; }
};

template <int WN, int B> struct Shape {
    static constexpr int kWR = kWaves / WN, kN = 32 * WN, kK = 32 * B, kRows = 32 * kWR;
    using OfN = Operand<kRows, kN>;
    using OfK = Operand<kRows, kK>;
    static constexpr int kA = OfN::kBlocks, kB = OfK::kBlocks;            // of a stage
    static_assert(kA == 2 * kWaves, "two a wavefront");
    static constexpr int kStage = (kA + kB) * kBlock, kPitch = pitch_of(B), kTurnedPitch = kN + 4;
    static constexpr int kGroupsK = kK / kKeptGroup, kGroups = kRows * kGroupsK, kHeld = (kGroups + kThreads - 1) / kThreads;
};

template <int WN, int B, bool kKept>
__global__ __launch_bounds__(kThreads, B == 5 ? 2 : 4) void kept_grad_kernel(GradArgs a)
{
    using L = Shape<WN, B>;
    extern __shared__ __align__(16) char smem[];
    // workgroups b, b + 8, .. run on one XCD: those of the same rows
    const int id = static_cast<int>(blockIdx.x), spread = a.splits >= 8;
    const int split = spread ? id % 8 + 8 * (id / 8 / a.tiles) : id / a.tiles, tile = spread ? id / 8 % a.tiles : id % a.tiles;
    if (split >= a.splits) return;
    const int n0 = tile / a.tiles_k * L::kN, k0 = tile % a.tiles_k * L::kK, N = a.N, K = a.K;
    const int64_t begin = split * a.rows, end = min(begin + a.rows, a.M);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave_n = wave % WN, wave_r = wave / WN, r32 = lane & 31, half = lane >> 5;
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem));

    // the piece of a block whose place is this lane, where it lies behind the first row of a stage; columns of the last tile that an operand has
    // not are any that it has: of results that nobody stores
    using OfN = typename L::OfN;
    using OfK = typename L::OfK;
    auto offset_of = [&](auto operand, int width, int first_column, int block) {
        using O = decltype(operand);
        return static_cast<uint32_t>((block / O::kAcross * O::kTall + O::row_at(lane)) * width +
                                     min(first_column + block % O::kAcross * O::kWide + 8 * O::piece_at(lane), width - 8)) * 2;
    };
    constexpr int kOwnK = kKept ? 1 : (L::kB + kWaves - 1) / kWaves;
    uint32_t offset_n[2], offset_k[kOwnK];
#pragma unroll
    for (int i = 0; i < 2; ++i) offset_n[i] = offset_of(OfN{}, N, n0, wave + i * kWaves);
#pragma unroll
    for (int i = 0; i < kOwnK; ++i) offset_k[i] = offset_of(OfK{}, K, k0, min(wave + i * kWaves, L::kB - 1));
    auto stage_block = [&](const void *rows, uint32_t offset, int row, int at, int left) {
        if (left >= L::kRows) {
            load_to_lds_from(lds + at, rows, offset);
        } else {
            half8 v = {};
            if (row < left) v = *reinterpret_cast<const half8 *>(static_cast<const char *>(rows) + offset);
            reinterpret_cast<half8 *>(smem + at)[lane] = v;
        }
    };
    // the next stage's codes, a group a thread and turn
    constexpr int kHeld = kKept ? L::kHeld : 1;
    uint4 held[kHeld];
    uint32_t held_bytes[kHeld], offset_codes[kHeld], offset_bytes[kHeld];
    if constexpr (kKept) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int g = min(tid + i * kThreads, L::kGroups - 1), column = min(k0 + g % L::kGroupsK * kKeptGroup, K - kKeptGroup);
            offset_codes[i] = static_cast<uint32_t>(g / L::kGroupsK * K + column);
            offset_bytes[i] = offset_codes[i] / kKeptGroup;
        }
    }
    const uint8_t *const codes = static_cast<const uint8_t *>(a.k), *const bytes = codes + a.M * K;
    auto fetch_codes = [&](int64_t row) {
        if (row >= end) return;
        const uint8_t *from = codes + row * K, *from_bytes = bytes + row * (K / kKeptGroup);
        const int left = static_cast<int>(min(end - row, static_cast<int64_t>(L::kRows)));
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const bool there = left >= L::kRows || min(tid + i * kThreads, L::kGroups - 1) / L::kGroupsK < left;
            held[i] = there ? *reinterpret_cast<const uint4 *>(from + offset_codes[i]) : make_uint4(0, 0, 0, 0);
            held_bytes[i] = there ? from_bytes[offset_bytes[i]] : 0;
        }
    };
    auto put_codes = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int g = tid + i * kThreads, r = g / L::kGroupsK, p = g % L::kGroupsK * 2;
            if (g >= L::kGroups) continue;
            half8 *to = reinterpret_cast<half8 *>(smem + buffer * L::kStage + (L::kA + r / OfK::kTall * OfK::kAcross + p / (OfK::kWide / 8)) * kBlock);
            const int r_in = r % OfK::kTall, p_in = p % (OfK::kWide / 8);
            to[OfK::place(r_in, p_in)] = kept_numbers(make_uint2(held[i].x, held[i].y), held_bytes[i]);
            to[OfK::place(r_in, p_in + 1)] = kept_numbers(make_uint2(held[i].z, held[i].w), held_bytes[i]);
        }
    };
    auto fetch = [&](int buffer, int64_t row) {
        const int left = static_cast<int>(min(end - row, static_cast<int64_t>(L::kRows)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = wave + i * kWaves;
            stage_block(a.n + row * N, offset_n[i], u / OfN::kAcross * OfN::kTall + OfN::row_at(lane), buffer * L::kStage + u * kBlock, left);
        }
        if constexpr (kKept) return;
#pragma unroll
        for (int i = 0; i < kOwnK; ++i) {
            const int u = wave + i * kWaves;
            if (u < L::kB)
                stage_block(static_cast<const _Float16 *>(a.k) + row * K, offset_k[i], u / OfK::kAcross * OfK::kTall + OfK::row_at(lane),
                            buffer * L::kStage + (L::kA + u) * kBlock, left);
        }
    };
    f32x16 acc[B];
    // dY's columns added up: by the workgroups of the first tile across; of the tile's columns by the wavefronts of its first rows
    constexpr int kSums = kKept ? 1 : B;
    float sums[kSums] = {};
#pragma unroll
    for (int j = 0; j < B; ++j) acc[j] = f32x16{};
    const bool sum_n = !a.turned && k0 == 0 && !a.sums, sum_k = a.turned && n0 == 0 && wave_n == 0;
    auto add_up = [](float &sum, const half8 &v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += static_cast<float>(v[e]);
    };
    const int asked_n = OfN::asked(lane, wave_n), asked_k[2] = {OfK::asked(lane, 0), OfK::asked(lane, 1)};
    auto column_of = [&](const char *from, int next) {
        typedef __attribute__((address_space(3))) lds_half4 *At;
        const auto *at = (__attribute__((address_space(3))) const char *)from;
        const lds_half4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((At)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((At)(at + next));
        const uint2 p = __builtin_bit_cast(uint2, lo), q = __builtin_bit_cast(uint2, hi);
        return __builtin_bit_cast(half8, make_uint4(p.x, p.y, q.x, q.y));
    };
    auto multiply = [&](int buffer) {
        const char *of_n = smem + buffer * L::kStage + asked_n, *of_k = smem + buffer * L::kStage + L::kA * kBlock;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const half8 n = column_of(of_n + OfN::start(2 * wave_r + s, wave_n), OfN::kNext);
            half8 k[B];
#pragma unroll
            for (int j = 0; j < B; ++j) k[j] = column_of(of_k + asked_k[j % 2] + OfK::start(2 * wave_r + s, j), OfK::kNext);
#pragma unroll
            for (int j = 0; j < B; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[j], n, acc[j], 0, 0, 0);
            if (sum_n) add_up(sums[0], n);
            if (!kKept && sum_k) {
#pragma unroll
                for (int j = 0; j < kSums; ++j) add_up(sums[j], k[j]);
            }
        }
    };
    int buffer = 0;
    if (kKept) fetch_codes(begin);
    fetch(0, begin);
    if (kKept) {
        put_codes(0);
        fetch_codes(begin + L::kRows);
    }
    for (int64_t row = begin; row < end; row += L::kRows, buffer ^= 1) {
        // the stage is there, and nobody reads the other buffer any more
        loads_done<0>();
        workgroup_barrier();
        if (row + L::kRows < end) {
            fetch(buffer ^ 1, row + L::kRows);
            if (kKept) {
                put_codes(buffer ^ 1);
                fetch_codes(row + 2 * L::kRows);
            }
        }
        multiply(buffer);
    }
    // the wavefronts' sums meet in LDS, those of one block of rows after the other, and leave as rows
    float *sum = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int w = 0; w < L::kWR; ++w) {
        __syncthreads();
        if (wave_r != w) continue;
        if (!a.turned) {
#pragma unroll
            for (int j = 0; j < B; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 *to = reinterpret_cast<f32x4 *>(sum + (wave_n * 32 + r32) * L::kPitch + 32 * j + 8 * g + 4 * half);
                    const f32x4 v = {acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]};
                    *to = w == 0 ? v : *to + v;
                }
        } else {
#pragma unroll
            for (int j = 0; j < B; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float *to = sum + (32 * j + e / 4 * 8 + 4 * half + e % 4) * L::kTurnedPitch + wave_n * 32 + r32;
                    *to = w == 0 ? acc[j][e] : *to + acc[j][e];
                }
        }
    }
    __syncthreads();
    float *part = a.parts + split * (static_cast<int64_t>(N) * K + (a.turned ? K : N));
    if (!a.turned) {
        for (int p = tid; p < L::kN * (L::kK / 4); p += kThreads) {
            const int n = p / (L::kK / 4), k = p % (L::kK / 4) * 4;
            if (n0 + n < N && k0 + k < K) *reinterpret_cast<f32x4 *>(part + static_cast<int64_t>(n0 + n) * K + k0 + k) = *reinterpret_cast<const f32x4 *>(sum + n * L::kPitch + k);
        }
    } else {
        for (int p = tid; p < L::kK * (L::kN / 4); p += kThreads) {
            const int k = p / (L::kN / 4), n = p % (L::kN / 4) * 4;
            if (n0 + n < N && k0 + k < K)
                *reinterpret_cast<f32x4 *>(part + static_cast<int64_t>(k0 + k) * N + n0 + n) = *reinterpret_cast<const f32x4 *>(sum + k * L::kTurnedPitch + n);
        }
    }
    // (the same for the whole workgroup)
    if (a.turned ? n0 != 0 : k0 != 0) return;
    if (a.sums) {
        constexpr int kShares = kThreads / L::kN;      // (a split's rows are whole groups of 32, but for the last one's)
        const int column = n0 + tid % L::kN;
        const int64_t last = (end + 31) / 32;
        float total = 0.0f;
#pragma unroll 8
        for (int64_t g = begin / 32 + tid / L::kN; g < last; g += kShares) total += a.sums[g * N + min(column, N - 1)];
        __syncthreads();
        sum[tid] = total;
        __syncthreads();
        if (tid >= L::kN || column >= N) return;
#pragma unroll
        for (int i = 1; i < kShares; ++i) total += sum[i * L::kN + tid];
        part[static_cast<int64_t>(N) * K + column] = total;
        return;
    }
    const int columns = a.turned ? L::kK : L::kN, first = a.turned ? k0 : n0, width = a.turned ? K : N;
#pragma unroll
    for (int j = 0; j < kSums; ++j) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sums[j]), __float_as_uint(sums[j]), false, false);
        sums[j] = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    }
#pragma unroll
    for (int w = 0; w < L::kWR; ++w) {
        __syncthreads();
        if (wave_r != w || half || (a.turned && wave_n)) continue;
#pragma unroll
        for (int j = 0; j < kSums; ++j) {
            if (j > 0 && !a.turned) continue;
            float *to = sum + (a.turned ? 32 * j : wave_n * 32) + r32;
            *to = w == 0 ? sums[j] : *to + sums[j];
        }
    }
    __syncthreads();
    if (tid < columns && first + tid < width) part[static_cast<int64_t>(N) * K + first + tid] = sum[tid];
}

// Tiles by what they pad, and the shares of the rows: as many as the chip has room for workgroups, but none of fewer than 256 rows.  The
// wider of two fp16 operands is the one whose columns are the tile's rows: it is read once where the other fits a tile's width.
constexpr int lds_of(int wn, int b)
{
    const int stages = 2 * (2 * kWaves + kWaves / wn * 2 * b) * kBlock, sums = 32 * wn * pitch_of(b) * 4, turned = 32 * b * (32 * wn + 4) * 4;
    return stages > sums && stages > turned ? stages : sums > turned ? sums : turned;
}

struct Plan {
    bool turned;
    int n, k, wn, b, tiles_k, tiles, splits;
    int64_t rows;
};

Plan plan_of(int64_t M, int N, int K, bool kept)
{
    auto padded = [](int width, int unit) { return (width + unit - 1) / unit * unit; };
    Plan p{};
    p.turned = !kept && K > N;
    p.n = p.turned ? K : N;
    p.k = p.turned ? N : K;
    p.wn = padded(p.n, 128) == padded(p.n, 64) ? 4 : 2;
    p.b = !kept && p.k <= 160 ? 5 : 4;
    for (int b : {4, 3, 2})
        if (padded(p.k, 32 * b) < padded(p.k, 32 * p.b)) p.b = b;
    p.tiles_k = padded(p.k, 32 * p.b) / (32 * p.b);
    p.tiles = padded(p.n, 32 * p.wn) / (32 * p.wn) * p.tiles_k;
    // (as many to an XCD as it has room for: one more would be a second round)
    const int step = 32 * kWaves / p.wn, room = p.b < 5 && 2 * lds_of(p.wn, p.b) <= 160 * 1024 ? 512 : 256;
    const int64_t most = ceil_div(M, 256), wanted = p.tiles * 8 <= room ? room / p.tiles / 8 * 8 : p.tiles < room ? room / p.tiles : 1;
    p.rows = ceil_div(ceil_div(M, most < wanted ? most : wanted), step) * step;
    p.splits = static_cast<int>(ceil_div(M, p.rows));
    return p;
}

template <int WN, int B> int launch(GradArgs a, bool kept, hipStream_t stream)
{
    using L = Shape<WN, B>;
    auto kernel = kept_grad_kernel<WN, B, false>;
    if constexpr (B < 5) kernel = kept ? kept_grad_kernel<WN, B, true> : kernel;
    constexpr int kLds = lds_of(WN, B);
    static_assert(kLds >= 2 * L::kStage && kLds >= L::kN * L::kPitch * 4 && kLds >= L::kK * L::kTurnedPitch * 4 && kLds <= 160 * 1024, "as the kernel uses it");
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), kLds)) return rc;
    const int64_t splits = a.splits >= 8 ? ceil_div(a.splits, 8) * 8 : a.splits;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(splits * a.tiles)), dim3(kThreads), kLds, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

}  // namespace

size_t kept_grads_bytes(const LinearGrad *grads, int num)
{
    size_t count = 0;
    for (int i = 0; i < num; ++i)
        count += static_cast<size_t>(plan_of(grads[i].M, grads[i].N, grads[i].K, grads[i].kept).splits) * (static_cast<size_t>(grads[i].N) * grads[i].K + grads[i].N);
    return count * sizeof(float);
}

int launch_kept_grad_parts(LinearGrad *grads, int num, float **parts, hipStream_t stream)
{
    for (int i = 0; i < num; ++i) {
        LinearGrad &g = grads[i];
        if (g.M < 1 || g.M > 0x7fffffff || g.N < 16 || g.N % 16 || g.K < 16 || g.K % 16 || g.N > 16384 || g.K > 16384)
            return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_linear_grad: M=%lld N=%d K=%d", (long long)g.M, g.N, g.K);
        const Plan p = plan_of(g.M, g.N, g.K, g.kept);
        if (g.sums && p.turned) return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_linear_grad: sums of %d columns beside %d", g.N, g.K);
        const GradArgs a{static_cast<const _Float16 *>(p.turned ? g.x : g.dy), p.turned ? g.dy : g.x, *parts, p.turned ? nullptr : g.sums, g.M, p.rows, p.n, p.k, p.tiles_k, p.tiles,
                         p.splits, p.turned};
        int rc = S3D_ERR_BAD_SHAPE;
        switch (p.wn * 8 + p.b) {
#define S3D_CASE(WN, B) case WN * 8 + B: rc = launch<WN, B>(a, g.kept, stream); break;
            S3D_CASE(2, 2) S3D_CASE(2, 3) S3D_CASE(2, 4) S3D_CASE(2, 5) S3D_CASE(4, 2) S3D_CASE(4, 3) S3D_CASE(4, 4) S3D_CASE(4, 5)
#undef S3D_CASE
        }
        if (rc) return rc;
        g.parts = *parts;
        g.splits = p.splits;
        *parts += static_cast<size_t>(p.splits) * (static_cast<size_t>(g.N) * g.K + g.N);
    }
    return S3D_OK;
}

}  // namespace s3d
