// The Swin blocks of a stage at inference (Swin3D/modules/swin3d_layers.py:563-625, 760-871) in one call.
//
// What bounds them on small scans is the host: through torch a block is some fifteen dispatches (300 us), while its seven
// kernels take a third of that.  Here the launches follow each other with nothing in between: per block
//   LayerNorm, qkv, attention, proj, add + LayerNorm, fc1 + GELU, fc2 (the last two as one on many rows)
// with the residual stream in fp32 and everything else in fp16, as under autocast.
#include "linear.h"

namespace s3d {
namespace {

bool fits(int64_t N, int32_t H, int32_t D, int32_t hidden, int32_t num_sets, int32_t num_blocks)
{
    return N >= 0 && H >= 1 && D >= 1 && H <= 1024 && D <= 1024 && H * D % 16 == 0 && H * D <= 1024 && hidden >= 16 && hidden % 16 == 0 && hidden <= 8192 &&
           num_sets >= 1 && num_blocks >= 1;
}

// in eight bits: rows behind a norm (in fp16 in front of an MLP in one kernel), or of the attention, with their scales, and q, k, v and the
// attention's result, or the MLP's scratch
struct EightBitPlaces {
    size_t scales, wide, total;
};

EightBitPlaces places_of(int64_t N, int32_t C, int32_t hidden)
{
    EightBitPlaces p{};
    const bool whole = mlp_pays(N, C, hidden);
    const size_t attention = static_cast<size_t>(N) * 4 * C * 2, mlp = whole ? 0 : s3d_mlp_int8_workspace_bytes(N, C, hidden);
    p.scales = align_up(static_cast<size_t>(N) * C * (whole ? 2 : 1), 256);
    p.wide = p.scales + align_up(static_cast<size_t>(N) * 4, 256);
    p.total = p.wide + align_up(attention > mlp ? attention : mlp, 256);
    return p;
}

// q, k, v and the attention's result side by side, then the hidden layer
size_t wide_bytes(int64_t N, int32_t C, int32_t hidden) { return align_up(static_cast<size_t>(N) * (hidden > 4 * C ? hidden : 4 * C) * 2, 256); }

}  // namespace
}  // namespace s3d

extern "C" __attribute__((visibility("default"))) size_t s3d_swin_blocks_workspace_bytes(int64_t N, int32_t C, int32_t hidden)
{
    using namespace s3d;
    if (N < 0 || C < 1 || hidden < 1) return 0;
    return align_up(static_cast<size_t>(N) * C * 2, 256) + wide_bytes(N, C, hidden);
}

extern "C" __attribute__((visibility("default"))) int s3d_swin_blocks(
    const float *x, float *x_out, void *pending, int64_t N, int32_t H, int32_t D, int32_t hidden, const int32_t *table_sizes,
    int32_t nd, int64_t table_len, const s3d_window_set *sets, int32_t num_sets, const s3d_swin_block *blocks,
    int32_t num_blocks, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace s3d;
    const int32_t C = H * D;
    if (N < 0 || H < 1 || D < 1 || C % 16 || C > 1024 || hidden < 16 || hidden % 16 || num_sets < 1 || num_blocks < 1)
        return fail(S3D_ERR_BAD_SHAPE, "s3d_swin_blocks: N=%lld H=%d D=%d hidden=%d (H D and hidden multiples of 16, H D at most "
                    "1024), %d sets, %d blocks", (long long)N, H, D, hidden, num_sets, num_blocks);
    if (N == 0) return S3D_OK;
    if (!x || !x_out || !pending || !table_sizes || !sets || !blocks)
        return fail(S3D_ERR_NULL_POINTER, "s3d_swin_blocks: null pointer");
    const size_t need = s3d_swin_blocks_workspace_bytes(N, C, hidden);
    if (!workspace || workspace_bytes < need)
        return fail(S3D_ERR_WORKSPACE, "s3d_swin_blocks: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *normed = static_cast<char *>(workspace), *wide = normed + align_up(static_cast<size_t>(N) * C * 2, 256);
    const size_t row = static_cast<size_t>(C) * 2;                  // bytes of C fp16 channels
    char *attended = wide + static_cast<size_t>(N) * 3 * row;       // behind q, k, v
    for (int i = 0; i < num_blocks; ++i) {
        const s3d_swin_block &b = blocks[i];
        const s3d_window_set &w = sets[i % num_sets];
        // (x itself stays as it is: from the first block's second sum on the stream is in x_out)
        const float *from = i == 0 ? x : x_out;
        if (int rc = s3d_add_layernorm(from, i == 0 ? nullptr : pending, S3D_DTYPE_F16, b.norm1_weight, b.norm1_bias, b.norm1_eps,
                                       i == 0 ? nullptr : x_out, normed, S3D_DTYPE_F16, N, C, stream))
            return rc;
        if (int rc = launch_linear({normed, b.qkv_weight, b.qkv_bias, wide, N, 3 * C, C, false}, s)) return rc;
        if (int rc = s3d_attn_fwd(wide, wide + row, wide + 2 * row, b.table_q, b.table_k, b.table_v, table_sizes, nd, table_len,
                                  w.w_sizes, w.w2n, w.n2n, w.n_coords, attended, nullptr, nullptr, N, H, D, w.num_windows, 3 * C,
                                  S3D_DTYPE_F16, w.planned ? S3D_ATTN_PLANNED : 0, w.plan, w.plan_bytes, stream))
            return rc;
        if (int rc = launch_linear({attended, b.proj_weight, b.proj_bias, pending, N, C, C, false}, s)) return rc;
        if (int rc = s3d_add_layernorm(from, pending, S3D_DTYPE_F16, b.norm2_weight, b.norm2_bias, b.norm2_eps, x_out, normed,
                                       S3D_DTYPE_F16, N, C, stream))
            return rc;
        if (mlp_pays(N, C, hidden)) {
            if (int rc = launch_mlp({normed, b.fc1_weight, b.fc1_bias, b.fc2_weight, b.fc2_bias, pending, N, C, hidden}, s)) return rc;
            continue;
        }
        if (int rc = launch_linear({normed, b.fc1_weight, b.fc1_bias, wide, N, hidden, C, true}, s)) return rc;
        if (int rc = launch_linear({wide, b.fc2_weight, b.fc2_bias, pending, N, C, hidden, false}, s)) return rc;
    }
    return S3D_OK;
}

// The same with the rows in front of every dense layer in eight bits: per block
//   norm, qkv, attention (in fp16, as q, k, v are), its rows in eight bits, proj, add + norm, and the MLP
// An MLP whose layers run as one kernel in fp16 (mlp.hip) stays that: us, fp16 / eight bits (mlp_int8.hip), hidden = 4 C, 14.2 / 17.3 at 20,000 rows of 80,
// 53.3 / 54.2 at 37,499 of 192, 101 / 144 at 149,993 of 160, 137 / 232 at 595,677 of 80, 185 / 228 at 200,000 of 192; with the norm ahead of it 19.4 / 23.3,
// 65.6 / 69.9, 151 / 193, 234 / 334, 259 / 301.  At the line (16,384 rows or 192 C), norm and MLP: 48 channels 12.0 / 12.3, 64 14.1 / 12.9, 80 18.3 / 16.0, 96 20.3 / 22.8, 128 29.3 / 29.8, 160 38.7 / 44.3,
// 192 64.4 / 69.7; at half of it eight bits take 0.72 to 1.05 of fp16's time, at twice 1.03 to 1.28.
extern "C" __attribute__((visibility("default"))) size_t s3d_swin_blocks_int8_workspace_bytes(int64_t N, int32_t C, int32_t hidden)
{
    using namespace s3d;
    if (C < 1 || C > 1024 || !fits(N, 1, C, hidden, 1, 1)) return 0;
    return places_of(N, C, hidden).total;
}

extern "C" __attribute__((visibility("default"))) int s3d_swin_blocks_int8(
    const float *x, float *x_out, void *pending, int64_t N, int32_t H, int32_t D, int32_t hidden, const int32_t *table_sizes,
    int32_t nd, int64_t table_len, const s3d_window_set *sets, int32_t num_sets, const s3d_swin_block_int8 *blocks,
    int32_t num_blocks, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace s3d;
    if (!fits(N, H, D, hidden, num_sets, num_blocks))
        return fail(S3D_ERR_BAD_SHAPE, "s3d_swin_blocks_int8: N=%lld H=%d D=%d hidden=%d (H D and hidden multiples of 16, at most 1024 and 8192), "
                    "%d sets, %d blocks", (long long)N, H, D, hidden, num_sets, num_blocks);
    if (N == 0) return S3D_OK;
    if (!x || !x_out || !pending || !table_sizes || !sets || !blocks) return fail(S3D_ERR_NULL_POINTER, "s3d_swin_blocks_int8: null pointer");
    const int32_t C = H * D;
    const EightBitPlaces p = places_of(N, C, hidden);
    if (!workspace || workspace_bytes < p.total)
        return fail(S3D_ERR_WORKSPACE, "s3d_swin_blocks_int8: workspace %zu B < required %zu B", workspace ? workspace_bytes : size_t(0), p.total);
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *base = static_cast<char *>(workspace), *wide = base + p.wide;
    int8_t *codes = reinterpret_cast<int8_t *>(base);
    float *scales = reinterpret_cast<float *>(base + p.scales);
    const size_t row = static_cast<size_t>(C) * 2;                  // bytes of C fp16 channels
    char *attended = wide + static_cast<size_t>(N) * 3 * row;       // behind q, k, v
    for (int i = 0; i < num_blocks; ++i) {
        const s3d_swin_block_int8 &b = blocks[i];
        const s3d_window_set &w = sets[i % num_sets];
        // (x itself stays as it is: from the first block's second sum on the stream is in x_out)
        const float *from = i == 0 ? x : x_out;
        if (int rc = s3d_add_norm_int8(from, i == 0 ? nullptr : pending, S3D_DTYPE_F16, b.norm1_weight, b.norm1_bias, b.norm1_eps, 0,
                                       i == 0 ? nullptr : x_out, codes, scales, N, C, stream))
            return rc;
        if (int rc = launch_linear_int8({codes, b.qkv_weight, scales, b.qkv_scales, b.qkv_bias, wide, N, 3 * C, C, false}, s)) return rc;
        if (int rc = s3d_attn_fwd(wide, wide + row, wide + 2 * row, b.table_q, b.table_k, b.table_v, table_sizes, nd, table_len,
                                  w.w_sizes, w.w2n, w.n2n, w.n_coords, attended, nullptr, nullptr, N, H, D, w.num_windows, 3 * C,
                                  S3D_DTYPE_F16, w.planned ? S3D_ATTN_PLANNED : 0, w.plan, w.plan_bytes, stream))
            return rc;
        if (int rc = launch_quantize_rows(attended, S3D_DTYPE_F16, codes, scales, N, C, s)) return rc;
        if (int rc = launch_linear_int8({codes, b.proj_weight, scales, b.proj_scales, b.proj_bias, pending, N, C, C, false}, s)) return rc;
        if (mlp_pays(N, C, hidden)) {
            if (int rc = s3d_add_layernorm(from, pending, S3D_DTYPE_F16, b.norm2_weight, b.norm2_bias, b.norm2_eps, x_out, base, S3D_DTYPE_F16, N, C, stream))
                return rc;
            if (int rc = launch_mlp({base, b.fc1_half, b.fc1_half_bias, b.fc2_half, b.fc2_half_bias, pending, N, C, hidden}, s)) return rc;
            continue;
        }
        if (int rc = s3d_add_norm_int8(from, pending, S3D_DTYPE_F16, b.norm2_weight, b.norm2_bias, b.norm2_eps, 0, x_out, codes, scales, N, C, stream))
            return rc;
        if (int rc = s3d_mlp_int8(codes, scales, b.fc1_weight, b.fc1_scales, b.fc1_bias, b.fc2_weight, b.fc2_scales, b.fc2_bias, pending, N, C, hidden, wide,
                                  p.total - p.wide, stream))
            return rc;
    }
    return S3D_OK;
}
