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

// exp and reciprocal as exact as T's results can show: fp32 takes the library's exp and v_rcp_f32 with a Newton
// step (1 + exp is 1 at least, so nothing but its overflow needs care; a third of a division's
// instructions), 16-bit types v_exp_f32 and v_rcp_f32 (within 2^-20 relative where sigmoid is not 0
// or 1).
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (sizeof(T) == 4) {
    const float y = 1.f + expf(-g), r = __builtin_amdgcn_rcpf(y);
    return y < 0x1p126f ? fmaf(fmaf(-y, r, 1.f), r, r) : r;
  } else {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  }
}

// The normal distribution's area below g, and its density.  In 16 bits the tail is e^(-g^2/2) t R(t) with t = 1
// / (1 + 0.6 |g| / sqrt(2)) and R of degree 7, fitted to erfcx(z) / t / 2 for z = |g| / sqrt(2) up
// to 10 (least largest relative error, 2^-21.6; with fp32's rounding 2^-19.9 up to |g| = 4): one exp
// for both, a third of erff's and expf's instructions.
template <typename T>
__device__ __forceinline__ void normal(float g, float* area, float* density) {
  if constexpr (sizeof(T) == 4) {
    *area = 0.5f + 0.5f * erff(g * 0.70710678f);
    *density = 0.39894228f * expf(-0.5f * g * g);
  } else {
    constexpr float R[8] = {0.169280037f, 0.168624625f,  0.145800158f, 0.0367074795f,
                            0.141881078f, -0.322222918f, 0.205969781f, -0.046040386f};
    const float t = __builtin_amdgcn_rcpf(fmaf(0.424264073f, fabsf(g), 1.f)), e = __builtin_amdgcn_exp2f(g * g * -0.72134752f);
    float r = R[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) r = fmaf(r, t, R[i]);
    const float tail = r * t * e;
    *area = g < 0.f ? tail : 1.f - tail;   // (NaN stays NaN)
    *density = 0.39894228f * e;
  }
}

// a = act(g), and its slope, of N elements: one switch for all of them, so that their chains of
// transcendentals interleave.
template <typename T, int N>
__device__ __forceinline__ void activate(int act, const float (&g)[N], float (&a)[N], float (&slope)[N]) {
  if (act == GSR_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = sigmoid<T>(g[i]);
      a[i] = g[i] * s;
      slope[i] = s * (1.f + g[i] * (1.f - s));
    }
  } else if (act == GSR_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float area, density;
      normal<T>(g[i], &area, &density);
      a[i] = g[i] * area;
      slope[i] = area + g[i] * density;
    }
  } else if (act == GSR_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = g[i] < 0.f ? 0.f : g[i];   // (NaN stays NaN)
      slope[i] = g[i] > 0.f ? 1.f : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = sigmoid<T>(g[i]);
      slope[i] = a[i] * (1.f - a[i]);
    }
  }
}

struct GatedShape {
  int64_t rows, dim, hidden;
};

// The projections g and u that a forward keeps for its backward, rows of gated_pad(hidden): fp32 as they
// are; of 16-bit blocks the upper 24 bits of their fp32 sums, in a plane of g's and u's upper
// halves and one of their next bytes (6 bytes an element; the truncation, 2^-16 at most, is a small
// part of the types' own half steps, where rounding g and u to the type would add as much again).
template <typename T>
struct Kept {
  uint32_t* hi;   // fp32: g
  uint16_t* lo;   // fp32: unused
  float* u;       // fp32: u
  __host__ __device__ Kept(void* p, int64_t rows, int64_t hidden) {
    const int64_t n = rows * gated_pad(hidden);
    hi = (uint32_t*)p;
    lo = (uint16_t*)(hi + n);
    u = (float*)(hi + n);
  }
  static int64_t bytes(int64_t rows, int64_t hidden) { return rows * gated_pad(hidden) * (sizeof(T) == 4 ? 8 : 6); }
  __device__ __forceinline__ void store(int64_t at, const float (&g)[8], const float (&v)[8]) const {   // at: a multiple of 8
    if constexpr (sizeof(T) == 4) {
      store_vec((float*)hi + at, g);
      store_vec(u + at, v);
    } else {
      uint32_t h[8], l[4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(g[i]), b = __float_as_uint(v[i]);
        h[i] = a >> 16 | (b & 0xFFFF0000u);
        const uint32_t next = (a >> 8 & 0xFFu) | (b & 0xFF00u);
        l[i / 2] = i % 2 ? l[i / 2] | next << 16 : next;
      }
      *(uint4*)(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
      *(uint4*)(hi + at + 4) = make_uint4(h[4], h[5], h[6], h[7]);
      *(uint4*)(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  }
  __device__ __forceinline__ void store_one(int64_t at, float g, float v) const {
    if constexpr (sizeof(T) == 4) {
      ((float*)hi)[at] = g;
      u[at] = v;
    } else {
      const uint32_t a = __float_as_uint(g), b = __float_as_uint(v);
      hi[at] = a >> 16 | (b & 0xFFFF0000u);
      lo[at] = (uint16_t)((a >> 8 & 0xFFu) | (b & 0xFF00u));
    }
  }
  __device__ __forceinline__ void load(int64_t at, float (&g)[8], float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
      load_vec((const float*)hi + at, g);
      load_vec(u + at, v);
    } else {
      const uint4 a = *(const uint4*)(hi + at), b = *(const uint4*)(hi + at + 4), c = *(const uint4*)(lo + at);
      const uint32_t h[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, l[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t next = i % 2 ? l[i / 2] >> 16 : l[i / 2];
        g[i] = __uint_as_float(h[i] << 16 | (next & 0xFFu) << 8);
        v[i] = __uint_as_float((h[i] & 0xFFFF0000u) | (next & 0xFF00u));
      }
    }
  }
};

}  // namespace gsr
