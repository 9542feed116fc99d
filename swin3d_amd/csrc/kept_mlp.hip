// Both layers of an MLP in training that keeps its inputs in eight bits, and the first half of their gradients, in one kernel each
// (gfx950; kept_rows.hip has the formulas, rows8.h the form):
//
//   forward    h = fp16(x W1^T + b1);  y = GELU(h) W2^T + b2;  x and h in eight bits
//   backward   dh = (dy W2) GELU'(h');  dx = dh W1;  dh and GELU(h') in fp16, for the weights' gradients
//
// Both are two products with what belongs to a hidden number between them, so both are the plan of mlp.hip: a wavefront takes 32 rows
// through both, 32 hidden channels at a time, which stay in registers between the products (the halves of each sixteen change places,
// v_permlane32_swap); weights come through LDS, the next ones on their way meanwhile.  A lane has numbers 8 g + 4 half .. + 3 of 32 hidden
// channels of its row; sixteen channels, a group of the kept form, are in a row's two lanes.
//
// Bound by instructions, of GELU, its derivative and the codes, and by what leaves: 149,993 rows of 160 over 640 forward 138 us (0.45 of 1.36 PFLOP/s, 1.6
// TB/s), backward 201 (3.0 TB/s; dh's sums in fp32 are 1 to 4% of the call), passes one after the other; the first twenty on an idle card take up to a fifth
// longer, 165 and 227, the forward without codes 25 less, and it is there that the backward's kernel was timed without its stores (below).
#include "attn_kernels.h"
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kRows = kThreads / 64 * 32;      // rows of a workgroup
constexpr int kHidden = 32, kMostHidden = 1024;                // hidden channels at a time, and of a layer

template <int C> struct Mlp {
    static_assert(C % 16 == 0, "steps of 16");
    static constexpr int kSteps = C / 16, kTiles = (C + 31) / 32;
    // LDS, in pieces of 16 bytes: rows of both weights an odd number of pieces apart, so that sixteen rows' pieces lie in all banks
    static constexpr int kPitch1 = C / 8 | 1, kPitch2 = kHidden / 8 + 1;
    static constexpr int kPieces = 8 * C, kLoads = (kPieces + kThreads - 1) / kThreads;
    static constexpr int kBuffer = kHidden * kPitch1 + C * kPitch2;
    static constexpr int kOutPitch = 32 + 8;                   // of 32 finished rows of 32 channels of a wavefront, in numbers
    static constexpr int kOut = kThreads / 64 * 32 * kOutPitch / 8;
    static constexpr int kLds = 2 * kBuffer > kOut ? 2 * kBuffer : kOut;
};

enum class Way { kPlain, kKeep, kBackward };      // kPlain: nothing behind the hidden layer has a gradient

template <int C, Way kWay>
__global__ __launch_bounds__(kThreads, 2) void kept_mlp_kernel(const KeptMlp a)
{
    constexpr bool kBackward = kWay == Way::kBackward, kKeep = kWay == Way::kKeep;
    using L = Mlp<C>;
    __shared__ __align__(16) half8 weights_s[L::kLds];
    __shared__ __align__(16) float bias_s[kBackward ? 4 : kMostHidden];
    __shared__ __align__(16) half8 hidden_s[kBackward ? kThreads / 64 * 2 * 32 * L::kOutPitch / 8 : 1];
    const _Float16 *x = static_cast<const _Float16 *>(a.x), *w1 = static_cast<const _Float16 *>(a.w1), *w2 = static_cast<const _Float16 *>(a.w2);
    const _Float16 *b1 = static_cast<const _Float16 *>(a.b1), *b2 = static_cast<const _Float16 *>(a.b2);
    const int M = static_cast<int>(a.M), hidden = a.hidden;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, half = lane >> 5;
    const int m0 = static_cast<int>(blockIdx.x) * kRows + wave * 32;
    // Lanes behind the last row do what its lanes do, stores of the same bits included: no branch around a store, behind which the compiler
    // would wait for all stores where it has to wait for loads.
    const int m = min(m0 + r32, M - 1);

    // this thread's pieces of the weights: of 32 rows of the first, which lie one after the other, and of 32 columns of the second
    const _Float16 *from[L::kLoads];
    int to[L::kLoads], ahead[L::kLoads];
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
        const int p = min(tid + i * kThreads, L::kPieces - 1), q = p - 4 * C;
        const bool first = q < 0;
        from[i] = first ? w1 + p * 8 : w2 + static_cast<int64_t>(q >> 2) * hidden + (q & 3) * 8;
        ahead[i] = first ? kHidden * C : kHidden;
        to[i] = first ? p / (C / 8) * L::kPitch1 + p % (C / 8) : kHidden * L::kPitch1 + (q >> 2) * L::kPitch2 + (q & 3);
    }
    // A stage is the first weights of 32 hidden channels and the second ones of those before them.  (No load behind a branch, where it
    // would be waited for at once: what there is none of comes again, and a thread without a piece has the last one.)
    half8 held[L::kLoads];
    const int chunks = hidden / kHidden;
    auto fetch = [&](int stage) {
#pragma unroll
        for (int i = 0; i < L::kLoads; ++i) {
            held[i] = *reinterpret_cast<const half8 *>(from[i]);
            from[i] += ahead[i] == kHidden ? (stage > 0 ? kHidden : 0) : (stage + 1 < chunks ? kHidden * C : 0);
        }
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < L::kLoads; ++i) weights_s[buffer * L::kBuffer + to[i]] = held[i];
    };
    // what is kept of the hidden layer: this lane's sixteen channels of a chunk, and the bytes of its two groups
    uint8_t *const codes_h = static_cast<uint8_t *>(a.kept_h) + static_cast<int64_t>(m) * hidden + 16 * half;
    uint8_t *const scales_h = static_cast<uint8_t *>(a.kept_h) + static_cast<int64_t>(M) * hidden + static_cast<int64_t>(m) * (hidden / kKeptGroup);
    uint4 codes, next_codes;
    uint32_t scales, next_scales;
    auto fetch_kept = [&](uint4 &c, uint32_t &s, int chunk) {
        c = *reinterpret_cast<const uint4 *>(codes_h + chunk * kHidden);
        s = *reinterpret_cast<const uint16_t *>(scales_h + chunk * 2);
    };
    fetch(0);
    if (kBackward) fetch_kept(codes, scales, 0);
    half8 rows[L::kSteps];
    {
        const _Float16 *row = x + static_cast<int64_t>(m) * C + 8 * half;
#pragma unroll
        for (int s = 0; s < L::kSteps; ++s) rows[s] = *reinterpret_cast<const half8 *>(row + 16 * s);
    }
    put(0);
    if (!kBackward)
        for (int t = tid; t < hidden; t += kThreads) bias_s[t] = b1 ? static_cast<float>(b1[t]) : 0.0f;
    f32x16 acc[L::kTiles];
#pragma unroll
    for (int j = 0; j < L::kTiles; ++j) acc[j] = f32x16{};
    // (the rows are there: a wait for them inside the loop would also be one for its own loads)
#pragma unroll
    for (int r = 0; r < L::kSteps; ++r) asm volatile("" : "+v"(rows[r]));
    auto both = [](uint32_t v, auto op) {
        const auto w = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return op(w[0], w[1]);
    };
    auto larger = [](uint32_t p, uint32_t q) { return max(p, q); };
    if (!kBackward && a.kept_x) {
        uint8_t *codes_x = static_cast<uint8_t *>(a.kept_x) + static_cast<int64_t>(m) * C + 8 * half;
        uint8_t *scales_x = static_cast<uint8_t *>(a.kept_x) + static_cast<int64_t>(M) * C + static_cast<int64_t>(m) * L::kSteps;
#pragma unroll
        for (int s = 0; s < L::kSteps; ++s) {
            const uint32_t byte = kept_byte(both(largest_bits(rows[s]), larger));
            const uint2 c = kept_codes(rows[s], Divisor(byte));
            *reinterpret_cast<uint2 *>(codes_x + 16 * s) = c;
            scales_x[s] = static_cast<uint8_t>(byte);
        }
    }
    __syncthreads();
    auto first_layer = [&](f32x16 &sum, int buffer, int begin, int end) {
        const half8 *at = weights_s + buffer * L::kBuffer + r32 * L::kPitch1 + half;
#pragma unroll
        for (int s = begin; s < end; ++s) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(at[2 * s], rows[s], sum, 0, 0, 0);
    };
    uint2 h[4], u[4];      // four numbers each: what the second layer takes, and what else leaves
    float summed[kBackward ? 16 : 1];
    const bool there = m0 + r32 < M;
    uint32_t word[4];
    auto activate = [&](const f32x16 &sum, int chunk, int g) {
        half4 o, v;
        if constexpr (kBackward) {
            const float s = kept_scale(g < 2 ? scales & 0xffu : scales >> 8);      // (rows behind the last one are copies of it, for the sums nothing)
            auto one = [&](int e, float code) {
                const Active at = gelu_and_slope(code * s);
                const float d = sum[4 * g + e] * at.slope;
                o[e] = to_half(d);
                v[e] = to_half(at.value);
                summed[4 * g + e] = there ? d : 0.0f;
            };
            one(0, code_of<0>(word[g]));
            one(1, code_of<1>(word[g]));
            one(2, code_of<2>(word[g]));
            one(3, code_of<3>(word[g]));
        } else {
            const f32x4 b = *reinterpret_cast<const f32x4 *>(bias_s + chunk * kHidden + 8 * g + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = to_half(sum[4 * g + e] + b[e]);
                o[e] = to_half(gelu(static_cast<float>(v[e])));
            }
        }
        h[g] = __builtin_bit_cast(uint2, o);
        u[g] = __builtin_bit_cast(uint2, v);
    };
    // the codes that the lane's chunk comes as, in order of g: words 2 g + half of its row's eight
    auto spread = [&]() {
        const auto a02 = __builtin_amdgcn_permlane32_swap(codes.x, codes.y, false, false), a13 = __builtin_amdgcn_permlane32_swap(codes.z, codes.w, false, false);
        word[0] = a02[0];
        word[2] = a02[1];
        word[1] = a13[0];
        word[3] = a13[1];
    };
    // forward: codes of a group, numbers 8 g + 4 half .. + 3 for g = 2 group and the one behind it
    uint32_t bytes = 0;
    auto keep_group = [&](int group) {
        const half4 p = __builtin_bit_cast(half4, u[2 * group]), q = __builtin_bit_cast(half4, u[2 * group + 1]);
        const uint32_t byte = kept_byte(both(largest_bits(half8{p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]}), larger));
        const Divisor d(byte);
        word[2 * group] = kept_codes(p, d);
        word[2 * group + 1] = kept_codes(q, d);
        bytes = bytes >> 8 | byte << 24;
    };
    auto store_kept = [&](int chunk) {
        const auto lo = __builtin_amdgcn_permlane32_swap(word[0], word[2], false, false), hi = __builtin_amdgcn_permlane32_swap(word[1], word[3], false, false);
        *reinterpret_cast<uint4 *>(codes_h + chunk * kHidden) = make_uint4(lo[0], lo[1], hi[0], hi[1]);
        *reinterpret_cast<uint16_t *>(scales_h + chunk * 2) = static_cast<uint16_t>(bytes >> 16);
    };
    // hidden channels 16 s + 8 half .. + 7
    auto joined = [&](const uint2 (&v)[4], int s) {
        const auto lo = __builtin_amdgcn_permlane32_swap(v[2 * s].x, v[2 * s + 1].x, false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(v[2 * s].y, v[2 * s + 1].y, false, false);
        return __builtin_bit_cast(half8, make_uint4(lo[0], hi[0], lo[1], hi[1]));
    };
    // The hidden layer's numbers leave 32 channels of a row at once, through the wavefront's own part of LDS (no barrier): in pieces of 32 bytes a row
    // the call takes 1.5 to 4% longer (149,993 rows of 160 over 640, us, 390 / 380, 595,677 of 80 over 320 636 / 612).  The stores cost what the
    // instructions do not hide: without them the kernel of 149,993 rows takes 133 of 228 us, without GELU and its derivative 206.
    _Float16 *const rows_s = reinterpret_cast<_Float16 *>(hidden_s) + wave * (2 * 32 * L::kOutPitch);
    auto stage_hidden = [&](const half8 &terms, int s) {
        _Float16 *at = rows_s + r32 * L::kOutPitch + 16 * s + 8 * half;
        *reinterpret_cast<half8 *>(at) = terms;
        *reinterpret_cast<half8 *>(at + 32 * L::kOutPitch) = joined(u, s);
    };
    float *const sums_at = kBackward ? a.sums + static_cast<int64_t>(min(m0, M - 1) / 32) * hidden + summed_column(lane) : nullptr;
    auto store_hidden = [&](int chunk) {
        if constexpr (kBackward) {
            const float sum = column_sum(summed, lane);
            if (m0 < M) sums_at[chunk * kHidden] = sum;      // (the same for the whole wavefront)
        }
        wave_fence();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = t * 16 + lane / 4, n = lane % 4 * 8;
            const int64_t to = static_cast<int64_t>(min(m0 + r, M - 1)) * hidden + chunk * kHidden + n;
            *reinterpret_cast<half8 *>(static_cast<_Float16 *>(a.dh) + to) = *reinterpret_cast<const half8 *>(rows_s + r * L::kOutPitch + n);
            *reinterpret_cast<half8 *>(static_cast<_Float16 *>(a.active) + to) = *reinterpret_cast<const half8 *>(rows_s + (32 + r) * L::kOutPitch + n);
        }
        wave_fence();
    };
    auto second_layer = [&](const half8 &terms, int s, int buffer, int begin, int end) {
        const half8 *at = weights_s + buffer * L::kBuffer + kHidden * L::kPitch1 + half;
#pragma unroll
        for (int j = begin; j < end; ++j) {
            const int r = 32 * j + 32 <= C ? 32 * j + r32 : min(32 * j + r32, C - 1);
            acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(at[r * L::kPitch2 + 2 * s], terms, acc[j], 0, 0, 0);
        }
    };
    fetch(1);
    if (kBackward) spread();
    f32x16 sum = {};
    first_layer(sum, 0, 0, L::kSteps);
    put(1);
    __syncthreads();
    for (int t = 1; t < chunks; ++t) {
        const int buffer = t & 1;
        fetch(t + 1);
        if (kBackward) fetch_kept(next_codes, next_scales, t);
        f32x16 next = {};
        half8 terms;
        // the hidden numbers' instructions between the products of the next hidden channels, then those of the second layer with the first
        // half of these
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            __builtin_amdgcn_sched_barrier(0);
            constexpr int kHalf = L::kSteps / 2, kSome = L::kTiles / 2;
            if (g == 2) terms = joined(h, 0);
            if (g < 2) first_layer(next, buffer, g == 0 ? 0 : kHalf, g == 0 ? kHalf : L::kSteps);
            else second_layer(terms, 0, buffer, g == 2 ? 0 : kSome, g == 2 ? kSome : L::kTiles);
            activate(sum, t - 1, g);
            if (kKeep && g % 2 == 1) keep_group(g / 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (kBackward) stage_hidden(terms, 0);
        terms = joined(h, 1);
        if (kBackward) stage_hidden(terms, 1);
        second_layer(terms, 1, buffer, 0, L::kTiles);
        if (kBackward) store_hidden(t - 1);
        if (kKeep) store_kept(t - 1);
        sum = next;
        if (kBackward) {
            codes = next_codes;
            scales = next_scales;
            spread();
        }
        put(buffer ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        activate(sum, chunks - 1, g);
        if (kKeep && g % 2 == 1) keep_group(g / 2);
    }
    if (kKeep) store_kept(chunks - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const half8 terms = joined(h, s);
        if (kBackward) stage_hidden(terms, s);
        second_layer(terms, s, chunks & 1, 0, L::kTiles);
    }
    if (kBackward) store_hidden(chunks - 1);
    __syncthreads();
    // the result leaves as rows, 32 channels at a time through the wavefront's own part of LDS (no barrier)
    _Float16 *out = reinterpret_cast<_Float16 *>(weights_s) + wave * (32 * L::kOutPitch), *y = static_cast<_Float16 *>(a.y);
#pragma unroll
    for (int j = 0; j < L::kTiles; ++j) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            half4 o, b = {0, 0, 0, 0};
            if (b2) b = *reinterpret_cast<const half4 *>(b2 + min(32 * j + 8 * g + 4 * half, C - 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = to_half(acc[j][4 * g + e] + static_cast<float>(b[e]));
            *reinterpret_cast<half4 *>(out + r32 * L::kOutPitch + 8 * g + 4 * half) = o;
        }
        wave_fence();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = t * 16 + lane / 4, n = lane % 4 * 8;
            const half8 v = *reinterpret_cast<const half8 *>(out + r * L::kOutPitch + n);
            if (m0 + r < M && (32 * j + 32 <= C || 32 * j + n < C)) *reinterpret_cast<half8 *>(y + static_cast<int64_t>(m0 + r) * C + 32 * j + n) = v;
        }
        wave_fence();
    }
}

template <int C, Way kWay> int launch(const KeptMlp &a, hipStream_t stream)
{
    hipLaunchKernelGGL((kept_mlp_kernel<C, kWay>), dim3(static_cast<unsigned>(ceil_div(a.M, kRows))), dim3(kThreads), 0, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

// (a kernel a width: its sums are so many registers.  The levels' widths of Swin3D-S and -L, 64 and 128; all others take two products.)
bool takes(int32_t C, int32_t hidden)
{
    const bool width = C == 48 || C == 64 || C == 80 || C == 96 || C == 128 || C == 160 || C == 192;
    return width && hidden >= kHidden && hidden % kHidden == 0 && hidden <= kMostHidden;
}

}  // namespace

// A workgroup has 128 rows and goes through all hidden channels: few rows leave CUs without work, the longer the more channels there are.
// us, two products / one kernel, hidden = 4 C: 16,384 rows of 48 17.4 / 14.9, of 96 23.1 / 25.1, 25,000 of 96 29.1 / 25.9, 20,000 of 128 30.3 / 33.5, 25,000
// of 128 37.6 / 33.3, of 160 43.7 / 39.9, 37,499 of 160 58.0 / 57.4, of 192 64.8 / 76.1, 60,000 of 192 95.0 / 79.4, 150,000 of 160 210 / 135, 200,000 of
// 192 334 / 261.
bool kept_mlp_pays(int64_t M, int32_t C, int32_t hidden) { return takes(C, hidden) && M >= 16384 && 3 * M >= 4 * C * C; }

// Here dh and GELU(h') leave either way, for the weights' gradients, so that it is only dh that is not read again, which GELU and its derivative,
// bound by instructions, do not make up for where there are many channels.  us, the backward's call, two products / one kernel: 16,384 rows of 48 35.7 / 33.7,
// of 80 45.2 / 45.3, 25,000 of 96 54.7 / 55.3, 37,499 of 80 59.0 / 61.9, 60,000 of 48 52.0 / 46.9, of 80 74.6 / 67.0, of 96 88.5 / 77.5, of 192 193 / 213,
// 200,000 of 192 617 / 649.  Of 128 and 160 channels as long as three quarters of what the chip has room for is at work (forward and backward together: 60,000
// of 160 228 / 216, 70,000 290 / 304, of 128 218 / 227, 149,993 of 160 543 / 535, 199,327 of 128 539 / 520, 300,000 of 160 1041 / 1024).
bool kept_mlp_grad_pays(int64_t M, int32_t C, int32_t hidden)
{
    if (!takes(C, hidden) || C > 160 || M < 16384) return false;
    const int64_t groups = ceil_div(M, kRows), room = 2 * static_cast<int64_t>(device_cus());
    return C <= 96 || 4 * groups >= 3 * room * ceil_div(groups, room);
}

int launch_kept_mlp(const KeptMlp &a, hipStream_t stream)
{
    switch (a.C) {
#define S3D_CASE(C) case C: return a.kept_h ? launch<C, Way::kKeep>(a, stream) : launch<C, Way::kPlain>(a, stream);
        S3D_CASE(48) S3D_CASE(64) S3D_CASE(80) S3D_CASE(96) S3D_CASE(128) S3D_CASE(160) S3D_CASE(192)
#undef S3D_CASE
    }
    return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_mlp: C=%d", a.C);
}

int launch_kept_mlp_grad(const KeptMlp &a, hipStream_t stream)
{
    switch (a.C) {
#define S3D_CASE(C) case C: return launch<C, Way::kBackward>(a, stream);
        S3D_CASE(48) S3D_CASE(64) S3D_CASE(80) S3D_CASE(96) S3D_CASE(128) S3D_CASE(160)
#undef S3D_CASE
    }
    return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_mlp_grad: C=%d", a.C);
}

}  // namespace s3d
