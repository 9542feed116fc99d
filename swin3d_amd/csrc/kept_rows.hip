// Dense layers in training that keep what their backward reads of their input in eight bits (gfx950); rows8.h has the form.
//
//   linear   y = x W^T + b;                       dx = dy W;  dW = dy^T x';  db = column sums of dy
//   MLP      h = x W1^T + b1;  y = GELU(h) W2^T + b2;
//            dh = (dy W2) GELU'(h');  dW2 = dy^T GELU(h');  dx = dh W1;  dW1 = dh^T x';  db2, db1 = column sums of dy, dh
//
// with x', h' what is kept of x and h (rounded to fp16).  Products of fp16 operands with sums in fp32; GELU(h') and dh are rounded to
// fp16 for the products behind them, which costs dx and dW1 as much again as their own rounding does (2.9 10^-4 of their norm for 2.1); db1 has no
// product behind it and is the sum of dh before it is rounded.  Of an MLP with hidden = 4 C that leaves 5.3 C bytes a row for the backward, where x, h and GELU(h)
// in fp16 are 18 C.
#include "linear.h"
#include "rows8.h"

namespace s3d {
namespace {

constexpr int kThreads = 256;

__host__ __device__ inline size_t codes_bytes(int64_t M, int32_t K) { return static_cast<size_t>(M) * K; }

// a group a thread; bound by memory (199,327 rows of 48 7.6 us, 3.9 TB/s)
__global__ __launch_bounds__(kThreads) void keep_kernel(const _Float16 *__restrict__ x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int64_t groups)
{
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < groups; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const half8 lo = reinterpret_cast<const half8 *>(x)[2 * i], hi = reinterpret_cast<const half8 *>(x)[2 * i + 1];
        const uint32_t byte = kept_byte(max(largest_bits(lo), largest_bits(hi)));
        const Divisor d(byte);
        const uint2 a = kept_codes(lo, d), b = kept_codes(hi, d);
        reinterpret_cast<uint4 *>(codes)[i] = make_uint4(a.x, a.y, b.x, b.y);
        scales[i] = static_cast<uint8_t>(byte);
    }
}

// GELU as the kernels have it that take its derivative too
__device__ __forceinline__ half8 gelu_of(const half8 &v)
{
    half8 u;
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = to_half(gelu_and_slope(v[e]).value);
    return u;
}

// half a group a thread: what the codes stand for to `out`, GELU of it to `active`; either may be null
__global__ __launch_bounds__(kThreads) void kept_values_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, _Float16 *__restrict__ out,
                                                               _Float16 *__restrict__ active, int64_t pieces)
{
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const half8 v = kept_numbers(reinterpret_cast<const uint2 *>(codes)[i], scales[i / 2]);
        if (out) reinterpret_cast<half8 *>(out)[i] = v;
        if (active) reinterpret_cast<half8 *>(active)[i] = gelu_of(v);
    }
}

// Parameters as the products read them: fp16 copies of those in fp32, and transposed ones of weights.  Tiles of 64 x 64 that turn in LDS;
// a bias is a matrix of one row.  One launch for all copies of a call (4 to 5 us for weights of up to 640 x 160, bound by it; 6 to 8, at times 12, for 1152 x 384
// in fp32, both copies of which are 3.5 MB to read and write).
constexpr int kSquare = 64, kMostCopies = 4;
struct Copies {
    const void *from[kMostCopies];
    _Float16 *to[kMostCopies], *turned[kMostCopies];      // either may be null
    int rows[kMostCopies], cols[kMostCopies], first[kMostCopies];
    int64_t scaled[kMostCopies];                          // that many numbers are multiplied by `scale`, in fp32
    bool half[kMostCopies];
    int num, blocks;
    float scale;

    // adds `from` where anything is wanted of it; what the products read of it
    const void *add(const void *array, int32_t dtype, int32_t r, int32_t c, void *copy, void *transposed, int64_t times_scale = 0)
    {
        const bool as_is = dtype == S3D_DTYPE_F16 && times_scale == 0;
        if (!array || (as_is && !transposed)) return array;
        from[num] = array;
        to[num] = as_is ? nullptr : static_cast<_Float16 *>(copy);
        turned[num] = static_cast<_Float16 *>(transposed);
        rows[num] = r;
        cols[num] = c;
        scaled[num] = times_scale;
        half[num] = dtype == S3D_DTYPE_F16;
        first[num++] = blocks;
        blocks += (r + kSquare - 1) / kSquare * ((c + kSquare - 1) / kSquare);
        return as_is ? array : copy;
    }
};

__global__ __launch_bounds__(kThreads) void copies_kernel(Copies a)
{
    __shared__ __align__(16) _Float16 tile_s[kSquare][kSquare + 4];
    int which = 0;
#pragma unroll
    for (int i = 1; i < kMostCopies; ++i) which = i < a.num && static_cast<int>(blockIdx.x) >= a.first[i] ? i : which;
    const void *from = a.from[0];
    _Float16 *to = a.to[0], *turned = a.turned[0];
    int rows = a.rows[0], cols = a.cols[0], first = a.first[0];
    int64_t scaled = a.scaled[0];
    bool half = a.half[0];
#pragma unroll
    for (int i = 1; i < kMostCopies; ++i) {
        if (which != i) continue;
        from = a.from[i]; to = a.to[i]; turned = a.turned[i]; rows = a.rows[i]; cols = a.cols[i]; first = a.first[i]; scaled = a.scaled[i]; half = a.half[i];
    }
    const int across = (cols + kSquare - 1) / kSquare, tile = static_cast<int>(blockIdx.x) - first, r0 = tile / across * kSquare, c0 = tile % across * kSquare;
    const int four = threadIdx.x % 16 * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = threadIdx.x / 16 + 16 * i;
        if (r0 + r >= rows || c0 + four >= cols) continue;
        const int64_t at = static_cast<int64_t>(r0 + r) * cols + c0 + four;
        half4 v;
        if (half) {
            v = *reinterpret_cast<const half4 *>(static_cast<const _Float16 *>(from) + at);
        } else {
            const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(from) + at);
            v = half4{static_cast<_Float16>(f.x), static_cast<_Float16>(f.y), static_cast<_Float16>(f.z), static_cast<_Float16>(f.w)};
            if (at < scaled) v = half4{to_half(f.x * a.scale), to_half(f.y * a.scale), to_half(f.z * a.scale), to_half(f.w * a.scale)};
        }
        if (half && at < scaled) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = to_half(static_cast<float>(v[e]) * a.scale);
        }
        if (to) *reinterpret_cast<half4 *>(to + at) = v;
        *reinterpret_cast<half4 *>(&tile_s[r][four]) = v;
    }
    if (!turned) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = threadIdx.x / 16 + 16 * i;
        if (c0 + c >= cols || r0 + four >= rows) continue;
        const half4 v = {tile_s[four][c], tile_s[four + 1][c], tile_s[four + 2][c], tile_s[four + 3][c]};
        *reinterpret_cast<half4 *>(turned + static_cast<int64_t>(c0 + c) * rows + r0 + four) = v;
    }
}

int launch_copies(const Copies &a, hipStream_t stream)
{
    if (a.blocks == 0) return S3D_OK;
    hipLaunchKernelGGL(copies_kernel, dim3(a.blocks), dim3(kThreads), 0, stream, a);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

bool is_dtype(int32_t d) { return d == S3D_DTYPE_F32 || d == S3D_DTYPE_F16; }
// room for the copies of a weight and a bias
size_t copies_bytes(int32_t N, int32_t K) { return align_up(2 * static_cast<size_t>(N) * K, 256) + align_up(2 * static_cast<size_t>(N), 256); }

dim3 grid_of(int64_t threads)
{
    const int64_t blocks = ceil_div(threads, kThreads);
    return dim3(static_cast<unsigned>(blocks < (1 << 22) ? blocks : 1 << 22));
}

bool rows_fit(int64_t M, int32_t K) { return M >= 0 && M <= 0x7fffffff && K >= 16 && K % 16 == 0 && K <= 16384; }
// (M = 0 has no gradients to speak of; the callers return zeros)
bool fits(int64_t M, int32_t N, int32_t K) { return rows_fit(M, K) && M >= 1 && N >= 16 && N % 16 == 0 && N <= 16384; }
bool scaled_fit(int32_t scaled, int32_t N) { return scaled >= 0 && scaled <= N && scaled % 16 == 0; }
int bad_shape(const char *who, int64_t M, int32_t N, int32_t K)
{
    return fail(S3D_ERR_BAD_SHAPE, "%s: M=%lld, widths %d and %d (M at least 1, widths multiples of 16, at most 16384)", who, (long long)M, K, N);
}

int keep(const void *x, void *kept, int64_t M, int32_t K, hipStream_t stream)
{
    uint8_t *codes = static_cast<uint8_t *>(kept);
    const int64_t groups = M * (K / kKeptGroup);
    hipLaunchKernelGGL(keep_kernel, grid_of(groups), dim3(kThreads), 0, stream, static_cast<const _Float16 *>(x), codes, codes + codes_bytes(M, K), groups);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

int values(const void *kept, void *out, void *active, int64_t M, int32_t K, hipStream_t stream)
{
    const uint8_t *codes = static_cast<const uint8_t *>(kept);
    const int64_t pieces = M * (K / 8);
    hipLaunchKernelGGL(kept_values_kernel, grid_of(pieces), dim3(kThreads), 0, stream, codes, codes + codes_bytes(M, K), static_cast<_Float16 *>(out),
                       static_cast<_Float16 *>(active), pieces);
    S3D_HIP_CHECK(hipGetLastError());
    return S3D_OK;
}

size_t linear_parts_bytes(int64_t M, int32_t N, int32_t K, bool kept)
{
    // (for the bias alone the other operand is any rows of 16 channels)
    LinearGrad g{nullptr, nullptr, nullptr, nullptr, M, N, K, 0, 1.0f}, bias{nullptr, nullptr, nullptr, nullptr, M, N, 16, 0, 1.0f};
    g.kept = kept;
    const size_t all = kept_grads_bytes(&g, 1), some = kept_grads_bytes(&bias, 1);
    return all > some ? all : some;
}

// GELU(h') and dh, dh's sums over each 32 rows, and the parts of the weights' gradients
struct MlpPlaces {
    size_t active, dhidden, sums, parts, total;
};
MlpPlaces mlp_places(int64_t M, int32_t C, int32_t hidden)
{
    MlpPlaces p{};
    const size_t wide = align_up(2 * codes_bytes(M, hidden), 256);
    p.dhidden = p.active + wide;
    p.sums = p.dhidden + wide;
    p.parts = p.sums + align_up(static_cast<size_t>(ceil_div(M, 32)) * hidden * 4, 256);
    p.total = p.parts + linear_parts_bytes(M, C, hidden, false) + linear_parts_bytes(M, hidden, C, true);
    return p;
}

}  // namespace
}  // namespace s3d

using namespace s3d;

extern "C" __attribute__((visibility("default"))) size_t s3d_kept_bytes(int64_t M, int32_t K)
{
    return rows_fit(M, K) ? codes_bytes(M, K) + codes_bytes(M, K) / kKeptGroup : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_keep_rows(const void *x, void *kept, int64_t M, int32_t K, void *stream)
{
    if (!rows_fit(M, K)) return fail(S3D_ERR_BAD_SHAPE, "s3d_keep_rows: M=%lld K=%d (K a multiple of 16, at most 16384)", (long long)M, K);
    if (M == 0) return S3D_OK;
    if (!x || !kept) return fail(S3D_ERR_NULL_POINTER, "s3d_keep_rows: null device pointer");
    return keep(x, kept, M, K, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) int s3d_kept_values(const void *kept, void *out, int64_t M, int32_t K, void *stream)
{
    if (!rows_fit(M, K)) return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_values: M=%lld K=%d (K a multiple of 16, at most 16384)", (long long)M, K);
    if (M == 0) return S3D_OK;
    if (!kept || !out) return fail(S3D_ERR_NULL_POINTER, "s3d_kept_values: null device pointer");
    return values(kept, out, nullptr, M, K, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) size_t s3d_kept_linear_workspace_bytes(int32_t N, int32_t K)
{
    return fits(1, N, K) ? copies_bytes(N, K) : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_kept_linear(const void *x, const void *w, int32_t w_dtype, const void *bias, int32_t bias_dtype,
                                                                      void *y, void *kept, void *w_t, int64_t M, int32_t N, int32_t K, int32_t scaled,
                                                                      float scale, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!fits(M, N, K)) return bad_shape("s3d_kept_linear", M, N, K);
    if (!scaled_fit(scaled, N)) return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_linear: %d scaled rows of %d (a multiple of 16)", scaled, N);
    if (!is_dtype(w_dtype) || (bias && !is_dtype(bias_dtype)))
        return fail(S3D_ERR_BAD_DTYPE, "s3d_kept_linear: dtypes %d, %d (0 = fp32, 1 = fp16)", w_dtype, bias_dtype);
    if (!x || !w || !y) return fail(S3D_ERR_NULL_POINTER, "s3d_kept_linear: null device pointer");
    const size_t need = copies_bytes(N, K);
    if (!workspace || workspace_bytes < need)
        return fail(S3D_ERR_WORKSPACE, "s3d_kept_linear: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *base = static_cast<char *>(workspace);
    Copies copies{};
    copies.scale = scale;
    w = copies.add(w, w_dtype, N, K, base, w_t, static_cast<int64_t>(scaled) * K);
    bias = copies.add(bias, bias_dtype, 1, N, base + align_up(2 * static_cast<size_t>(N) * K, 256), nullptr, scaled);
    if (int rc = launch_copies(copies, s)) return rc;
    if (kept)
        if (int rc = keep(x, kept, M, K, s)) return rc;
    return launch_linear({x, w, bias, y, M, N, K, false}, s);
}

extern "C" __attribute__((visibility("default"))) size_t s3d_kept_linear_grad_workspace_bytes(int64_t M, int32_t N, int32_t K)
{
    return fits(M, N, K) ? linear_parts_bytes(M, N, K, true) : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_kept_linear_grad(const void *dy, const void *w_t, const void *kept, void *dx, void *dw, void *db,
                                                                           int32_t grad_dtype, int64_t M, int32_t N, int32_t K, int32_t scaled,
                                                                           float scale, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!fits(M, N, K)) return bad_shape("s3d_kept_linear_grad", M, N, K);
    if (!scaled_fit(scaled, N)) return fail(S3D_ERR_BAD_SHAPE, "s3d_kept_linear_grad: %d scaled rows of %d (a multiple of 16)", scaled, N);
    if (grad_dtype != S3D_DTYPE_F32 && grad_dtype != S3D_DTYPE_F16)
        return fail(S3D_ERR_BAD_DTYPE, "s3d_kept_linear_grad: grad_dtype %d (0 = fp32, 1 = fp16)", grad_dtype);
    if (!dy || (dx && !w_t) || (dw && !kept)) return fail(S3D_ERR_NULL_POINTER, "s3d_kept_linear_grad: null device pointer");
    const size_t need = linear_parts_bytes(M, N, K, true);
    if (!workspace || workspace_bytes < need)
        return fail(S3D_ERR_WORKSPACE, "s3d_kept_linear_grad: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dx)
        if (int rc = launch_linear({dy, w_t, nullptr, dx, M, K, N, false}, s)) return rc;
    if (!dw && !db) return S3D_OK;
    LinearGrad g{dy, dw ? kept : dy, dw, db, M, N, dw ? K : 16, scaled, scale};
    g.kept = dw;
    float *parts = static_cast<float *>(workspace);
    if (int rc = launch_kept_grad_parts(&g, 1, &parts, s)) return rc;
    return launch_linear_grad_sums(&g, 1, nullptr, grad_dtype, s);
}

extern "C" __attribute__((visibility("default"))) size_t s3d_kept_mlp_workspace_bytes(int64_t M, int32_t C, int32_t hidden)
{
    if (!fits(M, hidden, C)) return 0;
    // copies of the parameters, and GELU of the hidden layer where the layers are two products
    return copies_bytes(hidden, C) + copies_bytes(C, hidden) + (kept_mlp_pays(M, C, hidden) ? 0 : align_up(2 * codes_bytes(M, hidden), 256));
}

extern "C" __attribute__((visibility("default"))) int s3d_kept_mlp(const void *x, const void *w1, const void *b1, const void *w2, const void *b2,
                                                                   const int32_t *dtypes, void *y, void *kept_x, void *kept_h, void *w1_t, void *w2_t,
                                                                   int64_t M, int32_t C, int32_t hidden, void *workspace, size_t workspace_bytes,
                                                                   void *stream)
{
    if (!fits(M, hidden, C)) return bad_shape("s3d_kept_mlp", M, hidden, C);
    if (!x || !w1 || !w2 || !y || !dtypes) return fail(S3D_ERR_NULL_POINTER, "s3d_kept_mlp: null pointer");
    for (int i = 0; i < 4; ++i)
        if (!is_dtype(dtypes[i])) return fail(S3D_ERR_BAD_DTYPE, "s3d_kept_mlp: dtype %d (0 = fp32, 1 = fp16)", dtypes[i]);
    const size_t need = s3d_kept_mlp_workspace_bytes(M, C, hidden);
    if (!workspace || workspace_bytes < need)
        return fail(S3D_ERR_WORKSPACE, "s3d_kept_mlp: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *base = static_cast<char *>(workspace);
    const size_t whole = align_up(2 * static_cast<size_t>(hidden) * C, 256);
    Copies copies{};
    w1 = copies.add(w1, dtypes[0], hidden, C, base, w1_t);
    b1 = copies.add(b1, dtypes[1], 1, hidden, base + whole, nullptr);
    base += copies_bytes(hidden, C);
    w2 = copies.add(w2, dtypes[2], C, hidden, base, w2_t);
    b2 = copies.add(b2, dtypes[3], 1, C, base + whole, nullptr);
    base += copies_bytes(C, hidden);
    if (int rc = launch_copies(copies, s)) return rc;
    if (kept_mlp_pays(M, C, hidden)) return launch_kept_mlp({x, w1, b1, w2, b2, y, kept_x, kept_h, nullptr, nullptr, nullptr, M, C, hidden}, s);
    if (kept_x)
        if (int rc = keep(x, kept_x, M, C, s)) return rc;
    LinearArgs first{x, w1, b1, base, M, hidden, C, false};
    first.keep = true;
    first.kept = kept_h;
    first.gelu_out = base;
    if (int rc = launch_linear(first, s)) return rc;
    return launch_linear({base, w2, b2, y, M, C, hidden, false}, s);
}

extern "C" __attribute__((visibility("default"))) size_t s3d_kept_mlp_grad_workspace_bytes(int64_t M, int32_t C, int32_t hidden)
{
    return fits(M, hidden, C) ? mlp_places(M, C, hidden).total : 0;
}

extern "C" __attribute__((visibility("default"))) int s3d_kept_mlp_grad(const void *dy, const void *w1_t, const void *w2_t, const void *kept_x,
                                                                        const void *kept_h, void *dx, void *dw1, void *db1, void *dw2, void *db2,
                                                                        int32_t grad_dtype, int64_t M, int32_t C, int32_t hidden, void *workspace,
                                                                        size_t workspace_bytes, void *stream)
{
    if (!fits(M, hidden, C)) return bad_shape("s3d_kept_mlp_grad", M, hidden, C);
    if (grad_dtype != S3D_DTYPE_F32 && grad_dtype != S3D_DTYPE_F16)
        return fail(S3D_ERR_BAD_DTYPE, "s3d_kept_mlp_grad: grad_dtype %d (0 = fp32, 1 = fp16)", grad_dtype);
    const bool behind = dx || dw1 || db1;      // the gradients behind that of the hidden layer
    if (!dy || ((behind || dw2) && !kept_h) || (behind && !w2_t) || (dx && !w1_t) || (dw1 && !kept_x))
        return fail(S3D_ERR_NULL_POINTER, "s3d_kept_mlp_grad: null device pointer");
    const MlpPlaces p = mlp_places(M, C, hidden);
    if (!workspace || workspace_bytes < p.total)
        return fail(S3D_ERR_WORKSPACE, "s3d_kept_mlp_grad: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), p.total);
    char *base = static_cast<char *>(workspace), *active = base + p.active, *dhidden = base + p.dhidden;
    float *sums = reinterpret_cast<float *>(base + p.sums);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!behind && dw2)
        if (int rc = values(kept_h, nullptr, active, M, hidden, s)) return rc;
    LinearGrad grads[2];
    int num = 0;
    if (dw2 || db2) grads[num++] = LinearGrad{dy, dw2 ? active : dy, dw2, db2, M, C, dw2 ? hidden : 16, 0, 1.0f};
    if (behind) {
        if (dx && kept_mlp_grad_pays(M, C, hidden)) {
            const KeptMlp a{dy, w2_t, nullptr, w1_t, nullptr, dx, nullptr, const_cast<void *>(kept_h), dhidden, active, sums, M, C, hidden};
            if (int rc = launch_kept_mlp_grad(a, s)) return rc;
        } else {
            LinearArgs a{dy, w2_t, nullptr, dhidden, M, hidden, C, false};
            a.kept_grad = true;
            a.kept = const_cast<void *>(kept_h);
            a.gelu_out = active;
            a.sums = sums;
            if (int rc = launch_linear(a, s)) return rc;
            if (dx)
                if (int rc = launch_linear({dhidden, w1_t, nullptr, dx, M, C, hidden, false}, s)) return rc;
        }
    }
    if (dw1 || db1) {
        grads[num] = LinearGrad{dhidden, dw1 ? kept_x : dhidden, dw1, db1, M, hidden, dw1 ? C : 16, 0, 1.0f};
        grads[num].kept = dw1;
        grads[num++].sums = sums;
    }
    if (num == 0) return S3D_OK;
    float *parts = reinterpret_cast<float *>(base + p.parts);
    if (int rc = launch_kept_grad_parts(grads, num, &parts, s)) return rc;
    return launch_linear_grad_sums(grads, num, nullptr, grad_dtype, s);
}
