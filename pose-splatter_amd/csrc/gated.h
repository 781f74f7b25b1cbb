// What the gated block's kernels share: the activations, and the epilogues that turn the two
// projections' fp32 sums into the block's output or into the gradients of both projections.
#pragma once

#include "types.h"

namespace gsr {

// Gradients of the two projections of a row lie side by side, [dg | pad | du | pad], each part
// padded with zeros to a multiple of kGatedPad columns: the products that read them take K in
// whole steps, and both weight gradients come from one product.
constexpr int kGatedPad = 64;
__host__ __device__ inline int64_t gated_pad(int64_t hidden) {
  return (hidden + kGatedPad - 1) / kGatedPad * kGatedPad;
}

// exp and reciprocal as exact as T's results can show: fp32 takes the library's, 16-bit types the
// hardware's v_exp_f32 and v_rcp_f32 (within 2^-20 relative where sigmoid is not 0 or 1).
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (sizeof(T) == 4) {
    return 1.f / (1.f + expf(-g));
  } else {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  }
}

// a = act(g), and its slope.
template <typename T>
__device__ __forceinline__ void activate(int act, float g, float& a, float& slope) {
  if (act == GSR_ACT_SILU) {
    const float s = sigmoid<T>(g);
    a = g * s;
    slope = s * (1.f + g * (1.f - s));
  } else if (act == GSR_ACT_GELU) {
    const float area = 0.5f + 0.5f * erff(g * 0.70710678f);
    a = g * area;
    slope = area + g * (0.39894228f * expf(-0.5f * g * g));
  } else if (act == GSR_ACT_RELU) {
    a = g < 0.f ? 0.f : g;   // (NaN stays NaN)
    slope = g > 0.f ? 1.f : 0.f;
  } else {
    a = sigmoid<T>(g);
    slope = a * (1.f - a);
  }
}

struct GatedShape {
  int64_t rows, dim, hidden;
};

}  // namespace gsr
