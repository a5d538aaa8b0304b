// What the kernels of a dense layer (ash_linear.hip, compiled once for every type of
// operands) and its C ABI (ash_layers.hip) share.
#pragma once

#include "ash_table.h"

#include "../../include/ash_hip.h"

namespace ash {

// One product  out[r, c] = sum_k P[r, k] Q[c, k]  and what becomes of it.
//   forward      P = input (rows x in),   Q = weight (out x in)
//   grad input   P = gz (rows x out),     Q = weight transposed (in x out)
//   grad weight  P = gz transposed (out x rows), Q = input transposed (in x rows)
// with gz = grad * slope, formed as the operand is read.
struct LinearJob {
    const void* input;
    const void* weight;
    const void* bias;
    const void* residual;
    const void* grad;         // gradients only: of the output
    const void* slope;        // f'(z) / slope_factor as the forward left it, or null: one
    float slope_factor;
    int32_t slope_kind;       // ash_linear.hip: SlopeKind
    const float* input_scales;
    const float* weight_scales;
    void* out;
    void* slope_out;
    int64_t rows, in, cols;   // cols: out features
    int64_t input_stride, residual_stride;
    int32_t out_dtype, activation;
    float act_scale;
    // second order: the gradient of the gradient of the input, an addend, and where t grad
    // f''(z) goes; `out` takes the gradient of `grad`
    const void* second_input;
    const void* addend;
    int64_t addend_stride;
    void* curvature_out;
    // weight's gradient: a second pair of operands whose product is added
    const void* second_grad;
    const void* second_slope;
    const void* second_factor;
    int64_t second_stride;
    bool second_has_bias;     // which pair's grad the bias' gradient sums
    void* weight_out;         // of the weight's gradient (`out`: the input's)
    void* bias_out;
    void* scratch;
    int32_t splits;           // parts the rows are cut into, per pair
};

enum LinearKind { kLinearForward, kLinearGradInput, kLinearGradWeight, kLinearSecond, kLinearGradBoth };

// Defined in ash_linear.hip, one set for every type.
template <int DTYPE>
int linear_run(LinearKind kind, const LinearJob& job, hipStream_t s);

// The tile of a weight's gradient (out x in): those of direct loads where 16-byte pieces and
// more than 64 features allow them; else 64 x 64 in 16 bits (40 000 rows of 131 fp16 to 257:
// 49 us, by 128 x 64 76, by 128 x 128 99); in float32 twice as high (65 536 rows of 512 to
// 512: 463 us, 64 x 64 538) unless that adds half a tile of nothing (of 131 to 257: 119 us
// for 153; of 67 to 129 10 007 rows 20 for 28, 40 000 58 for 47).
struct WeightTile {
    int rows, cols;
};
inline WeightTile weight_tile(int64_t in, int64_t out, int32_t dtype) {
    if (in <= 32) return {128, 32};
    if (out <= 64) return {64, 64};
    if (dtype == ASH_F32) return in > 64 && (out - 1) % 128 < 64 ? WeightTile{64, 64} : WeightTile{128, 64};
    if (in <= 64 || in % 8 != 0 || out % 8 != 0) return {64, 64};
    if (in > 512 && out > 512) return {256, 256};
    return {128, 128};
}

// Gradients of input and weight in one kernel: layers of up to 64 features in and out.
constexpr int64_t kNarrowFeatures = 64;
// Its workgroups (two a CU), each of which leaves a part of the weight's gradient.
inline int64_t narrow_backward_parts(int64_t rows, int pairs) {
    const int64_t slabs = (rows + 63) / 64 * pairs;
    return slabs < 512 ? slabs : 512;
}

// Parts that the rows are cut into for a weight's gradient (ash_layers.hip).
int32_t linear_splits(int64_t rows, int64_t in, int64_t out, int32_t dtype, int pairs);

}  // namespace ash
