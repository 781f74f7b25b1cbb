// Element types of the layer and optimizer kernels: fp32, bf16 and fp16 storage, fp32 arithmetic.
#pragma once

#include "gsr_common.h"

namespace gsr {

struct bf16 {
  uint16_t u;
};
struct f16 {
  _Float16 h;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float to_f(f16 v) { return (float)v.h; }

// To nearest, ties to even; NaN stays NaN (v_cvt_pk_bf16_f32 and v_cvt_f16_f32).
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) {
  return {__builtin_bit_cast(uint16_t, (__bf16)v)};
}
template <>
__device__ __forceinline__ f16 from_f<f16>(float v) { return {(_Float16)v}; }

// V consecutive elements moved as one access.  The target's global memory instructions take any
// byte address, so rows of odd lengths and strides keep 16-byte accesses.
template <typename T, int V>
struct __attribute__((packed)) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f(k.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// The first n of V elements (n <= 0: none); the others read as `fill` and are not written.
template <typename T, int V>
__device__ __forceinline__ void load_upto(const T* p, int64_t n, float (&out)[V], float fill = 0.f) {
  if (n >= V) {
    load_vec(p, out);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = i < n ? to_f(p[i]) : fill;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_upto(T* p, int64_t n, const float (&in)[V]) {
  if (n >= V) {
    store_vec(p, in);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = from_f<T>(in[i]);
  }
}

// 16 bytes of T as they lie in memory, four registers (an array of 16-bit elements would take eight),
// for loads that are to be in flight while others are worked on.  Elements from n on are zeros.
template <typename T>
struct Raw {
  static constexpr int V = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (__is_same(T, bf16)) {
      return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    } else {
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(i % 2 ? w[i / 2] >> 16 : w[i / 2]));
    }
  }
  __device__ __forceinline__ void load(const T* p, int64_t n) {
    if (n >= V) {
      const Pack<uint32_t, 4> k = *reinterpret_cast<const Pack<uint32_t, 4>*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = k.v[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4) {
          w[i] = __float_as_uint(p[i]);
        } else {
          w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i % 2));
        }
      }
  }
};

// A parameter vector (weights, biases) of type `type`, or `fill` where there is none.
template <int V>
__device__ __forceinline__ void load_param(const void* p, int type, int64_t at, int64_t n, float (&out)[V], float fill) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = fill;
  } else if (type == GSR_F32) {
    load_upto((const float*)p + at, n, out);
  } else if (type == GSR_BF16) {
    load_upto((const bf16*)p + at, n, out);
  } else {
    load_upto((const f16*)p + at, n, out);
  }
}

__device__ __forceinline__ void store_param(void* p, int type, int64_t at, float v) {
  if (type == GSR_F32) {
    ((float*)p)[at] = v;
  } else if (type == GSR_BF16) {
    ((bf16*)p)[at] = from_f<bf16>(v);
  } else {
    ((f16*)p)[at] = from_f<f16>(v);
  }
}

inline bool known_type(int t) { return t == GSR_F32 || t == GSR_BF16 || t == GSR_F16; }
inline size_t type_size(int t) { return t == GSR_F32 ? 4 : 2; }

}  // namespace gsr
