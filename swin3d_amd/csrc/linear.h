// Dense layers of fp16 rows (linear.hip).
#pragma once

#include "s3d_common.h"

namespace s3d {

struct LinearArgs {
    const void *x, *w, *bias;   // [M,K], [N,K], [N] or null; fp16
    void *y;                    // [M,N] fp16
    int64_t M;
    int32_t N, K;
    bool gelu;
    const void *gelu_at = nullptr;   // [M,N] fp16: the rows, rounded, are gradients behind a GELU of these, and y those before it
    bool in_order = false;           // a number's K products are added up one after the other, whatever the tile
    void *gelu_out = nullptr;        // [M,N] fp16: GELU of y's rounded rows, beside them (in_order; without gelu and gelu_at)
    // Rows in eight bits (rows8.h; without gelu, gelu_at and in_order, N a multiple of 16).  keep: in place of y the rounded rows go to kept
    // (unless it is null) and GELU of them to gelu_out.  kept_grad: the rows are gradients behind a GELU of what kept has, y those before it,
    // gelu_out GELU of what is kept, and sums the results added up over each 32 rows before they are rounded; no bias.
    bool keep = false, kept_grad = false;
    void *kept = nullptr;            // written by keep, read by kept_grad
    float *sums = nullptr;           // [ceil(M / 32)][N]
};

int launch_linear(const LinearArgs &a, hipStream_t stream);

// Both layers of an MLP in one kernel (mlp.hip): y = fc2(GELU(fc1(x)))
struct MlpArgs {
    const void *x, *w1, *b1, *w2, *b2;   // [M,C], [hidden,C], [hidden] or null, [C,hidden], [C] or null; fp16
    void *y;                             // [M,C] fp16, apart from x
    int64_t M;
    int32_t C, hidden;
};
bool mlp_takes(int64_t M, int32_t C, int32_t hidden);
bool mlp_pays(int64_t M, int32_t C, int32_t hidden);      // ... and is faster than the layers apart
int launch_mlp(const MlpArgs &a, hipStream_t stream);

// Both layers of an MLP of such rows as one kernel (mlp_int8.hip), where that is faster than the layers apart
struct MlpInt8 {
    const int8_t *x, *w1, *w2;                  // [M,C], [hidden,C], [C,hidden]
    const float *sx, *s1, *b1, *s2, *b2;        // [M], [hidden], [hidden] or null, [C], [C] or null
    void *y;                                    // [M,C] fp16
    int64_t M;
    int32_t C, hidden;
};
bool mlp_int8_pays(int64_t M, int32_t C, int32_t hidden);
int launch_mlp_int8(const MlpInt8 &a, hipStream_t stream);

// Dense layers of rows in eight bits (linear_int8.hip)
struct LinearInt8 {
    const int8_t *x, *w;              // [M,K], [N,K]
    const float *sx, *sw, *bias;      // [M], [N], [N] or null
    void *y;                          // [M,N] fp16
    int64_t M;
    int32_t N, K;
    bool gelu;
};
int launch_linear_int8(const LinearInt8 &l, hipStream_t stream);
// Rows of fp32 or fp16 in eight bits with a scale each (norm_int8.hip)
int launch_quantize_rows(const void *x, int32_t dtype, int8_t *codes, float *scales, int64_t N, int32_t C, hipStream_t stream);

// Both layers of an MLP in training that keeps its inputs in eight bits, in one kernel each way (kept_mlp.hip)
struct KeptMlp {
    const void *x, *w1, *b1, *w2, *b2;   // forward: [M,C], [hidden,C], [hidden] or null, [C,hidden], [C] or null; fp16
    void *y;                             // [M,C]
    void *kept_x, *kept_h;               // written by the forward unless null; kept_h is read by the backward
    void *dh, *active;                   // backward, [M,hidden] fp16: the hidden layer's gradients, and GELU of what is kept
    float *sums;                         // ... [ceil(M / 32)][hidden]: the gradients' sums over each 32 rows, before they are rounded
    int64_t M;
    int32_t C, hidden;
};
bool kept_mlp_pays(int64_t M, int32_t C, int32_t hidden);          // that is faster than two products
bool kept_mlp_grad_pays(int64_t M, int32_t C, int32_t hidden);     // ... for dx and what the weights' gradients read
int launch_kept_mlp(const KeptMlp &a, hipStream_t stream);
int launch_kept_mlp_grad(const KeptMlp &a, hipStream_t stream);    // x is dy, w1 and w2 are w2 and w1 transposed, y is dx; no biases

// A layer's weight and bias gradients (linear_grad.hip): dw = dy^T x, db = the column sums of dy; the first `scaled` rows of
// the weight (and numbers of the bias) are parameters times `scale`
struct LinearGrad {
    const void *dy, *x;   // [M,N], [M,K] fp16
    void *dw, *db;        // [N,K], [N]; one of them may be null
    int64_t M;
    int32_t N, K, scaled;
    float scale;
    const float *parts = nullptr;   // where launch_linear_grad_parts has put them, and how many
    int32_t splits = 0;
    bool kept = false;              // x in eight bits (rows8.h), for launch_kept_grad_parts
    const float *sums = nullptr;    // [ceil(M / 32)][N], for the same: db is the sum of these, those of dy over each 32 rows before it was rounded
};

constexpr int kMostLinearGrads = 4;
// room for the parts of `num` layers, however they are grouped
size_t linear_grads_bytes(const LinearGrad *grads, int num);
// the parts of `num` layers of as many rows, to *parts and on, which is moved behind them
int launch_linear_grad_parts(LinearGrad *grads, int num, float **parts, hipStream_t stream);

// The same for layers that keep their input in eight bits, and of an MLP's hidden layer in fp16 (kept_grad.hip); N and K multiples of 16
size_t kept_grads_bytes(const LinearGrad *grads, int num);
int launch_kept_grad_parts(LinearGrad *grads, int num, float **parts, hipStream_t stream);

// The gradients of (sum, y) = (x + residual, LayerNorm(x + residual)) (layernorm.hip), those of the norm's parameters in parts
struct NormGrad {
    const float *parts;      // [count][2 C]: of the weight, of the bias
    float *dgamma, *dbeta;
    int32_t count, C;
};
size_t layernorm_grad_bytes(int64_t N, int32_t C);
int launch_layernorm_grad(const float *sum, const float *dsum, const void *dy, const float *gamma, float eps, float *dx, void *dresidual, NormGrad *norm,
                          int64_t N, int32_t C, float *parts, hipStream_t stream);

// the sums of the parts of `num` layers and, unless null, of a norm in one launch
int launch_linear_grad_sums(const LinearGrad *grads, int num, const NormGrad *norm, int32_t grad_dtype, hipStream_t stream);

}  // namespace s3d
