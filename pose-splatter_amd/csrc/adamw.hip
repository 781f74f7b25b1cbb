// One AdamW step over many tensors in one launch (per 56 tensors), moments in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: each element is read and written once (28 bytes with fp32 parameters and
// 32-bit moments, 16 with 8-bit ones).  28 M fp32 elements with 8-bit moments 80 us step after step
// (5.6 TB/s), 95 between other kernels; 101 M in bf16 with 32-bit ones 417 us, 5.35 TB/s.  The list
// of tensors travels in the kernel's arguments, so nothing is uploaded, kept or looked up by
// address, and a step can be captured in a graph.
// A workgroup takes 2048 elements of one tensor, found by a binary search over the tensors'
// first workgroups; a wave takes 256 of them at a time, four a lane (16-byte loads of fp32).
//
// 8-bit moments are held in blocks of 256 elements with one fp32 unit each (a wave's own block:
// its largest magnitude is one wave reduction):
//   mean   e4m3 code q, m = q * unit, unit = max|m| / 448
//   root   r = sqrt(v) = k 2^(e-1) * unit with k = 16..31 and e = 1..15 (code 16 e + k - 16), or
//          k = 0..15 for codes below 16; unit = max r / 507904.  The root halves v's range, so
//          eight bits keep a relative step of 1/32 or better over 31 * 2^14 : 16.
// They are rounded to nearest (ties to even), or without bias: up with the probability that
// makes the expected mean, and the expected square of the root, the values before rounding, so that a
// chain of steps follows the recursion of unrounded moments on average.  Rounded to nearest a change of less
// than half a code step (1/32 of a root, 1/16 of a mean) in one step is lost, however many steps make
// it, and b2 = 0.999 changes a root by 1/2000 a step.  The draws are a hash of the element's place and
// the step count: the same bits every run, in any list, captured or not.  28 M fp32
// elements: 93 us a step against 80, the vector instructions of the draws.
// A root that is not zero keeps a code that is not, in both (a vanished denominator would turn a
// small gradient into a huge step).  The parameters' update uses the new moments before they are rounded.  Everything is fp32 without contraction into
// fused multiply-adds, so that a moment's code does not depend on how the compiler fused it.
#include "types.h"

#pragma clang fp contract(off)

namespace gsr {

constexpr int kAdamTensors = 56;    // a launch's arguments stay below 4 KB
constexpr int kAdamChunk = 2048;    // elements a workgroup
constexpr int kAdamBlock = GSR_ADAMW_BLOCK;
constexpr float kMeanTop = 448.f, kRootTop = 507904.f;
constexpr float kUnitTiny = 0x1p-100f;   // blocks below hold zeros: their unit's inverse would overflow

struct AdamList {
  gsr_adamw_tensor t[kAdamTensors];
  uint32_t first[kAdamTensors + 1];   // first workgroup of each tensor; the last entry: the total
  int count;
  uint32_t skip;   // workgroups of the first tensor that earlier launches took
};

struct AdamScalars {
  float b1, c1, b2, c2, eps, keep, size, rbias;   // c = 1 - b; keep = 1 - lr wd; size = lr / (1 - b1^t)
};

// b^t for a whole t by squaring, in double.
__host__ __device__ inline double power(double b, int64_t t) {
  double r = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}

__host__ __device__ inline AdamScalars adam_scalars(const gsr_adamw_args& a, double lr, int64_t step) {
  AdamScalars s;
  s.b1 = (float)a.beta1;
  s.c1 = (float)(1.0 - a.beta1);
  s.b2 = (float)a.beta2;
  s.c2 = (float)(1.0 - a.beta2);
  s.eps = (float)a.eps;
  s.keep = (float)(1.0 - lr * a.weight_decay);
  s.size = (float)(lr / (1.0 - power(a.beta1, step)));
  s.rbias = (float)(1.0 / sqrt(1.0 - power(a.beta2, step)));
  return s;
}

// p, m, v of one element; root: sqrt(v).
__device__ __forceinline__ void adam_element(const AdamScalars& s, float g, float& p, float& m, float& v, float& root) {
  m = m * s.b1 + g * s.c1;
  v = v * s.b2 + (g * g) * s.c2;
  root = sqrtf(v);
  const float denom = root * s.rbias + s.eps;
  p = p * s.keep - m * s.size / denom;
}

__device__ __forceinline__ float root_value(uint32_t code, float unit) {
  const uint32_t e = code >> 4, up = (e > 1 ? e : 1) - 1;
  return (float)((code - up * 16) << up) * unit;
}

// q = r / unit in [0, kRootTop]: to five significant bits, ties to even.
__device__ __forceinline__ uint32_t root_code(float q) {
  if (q < 16.f) return (uint32_t)rintf(q);
  uint32_t u = __float_as_uint(q < kRootTop ? q : kRootTop);
  u += 0x3FFFFu + ((u >> 19) & 1u);
  return (u >> 19) - (131u << 4) + 16u;   // exponent 131 (16..31) is code 16
}

// A whole number's 32 bits mixed (two multiplications by the golden ratio's and the root of 2's fractions).
__device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x = (x ^ x >> 16) * 0x9E3779B9u;
  x = (x ^ x >> 15) * 0x6A09E667u;
  return x ^ x >> 16;
}

__device__ __forceinline__ float draw24(uint32_t x) { return (float)(x >> 8) * 0x1p-24f; }   // [0, 1)

// |q| <= kMeanTop to one of the two e4m3 values beside it: up where `draw` lies below q's share of the step.
__device__ __forceinline__ float mean_unbiased(float q, uint32_t draw) {
  const float a = fabsf(q);
  float v;
  if (a < 0x1p-6f) {   // steps of 2^-9
    v = floorf(a * 0x1p9f + draw24(draw)) * 0x1p-9f;
  } else {             // three bits behind the first
    v = __uint_as_float((__float_as_uint(a) + (draw >> 12)) & 0xFFF00000u);
  }
  return q == q ? copysignf(v, q) : q;
}

// q in [0, kRootTop] to one of the two codes beside it, k and k + 1 steps: up with the probability (q^2 -
// k^2) / (2 k + 1) in steps, so that the square's expectation is q^2.
__device__ __forceinline__ uint32_t root_unbiased(float q, uint32_t draw) {
  const uint32_t u = __float_as_uint(q < kRootTop ? q : kRootTop);
  const bool low = q < 16.f;
  const float s = low ? q : __uint_as_float((u & 0x7FFFFFu) | 131u << 23);   // in steps: 16 to 32, or below
  const float k = floorf(s), f = s - k;
  const uint32_t code = (low ? 0u : ((u >> 23) - 131u) * 16u) + (uint32_t)k;
  return code + (draw24(draw) * (2.f * k + 1.f) < f * (2.f * k + f) ? 1u : 0u);
}

// Largest of 64 lanes' bit patterns: magnitudes order as integers, NaN above all.
__device__ __forceinline__ float wave_max_abs(float a, float b, float c, float d) {
  const int x = gsr_max_i(__float_as_int(fabsf(a)), __float_as_int(fabsf(b)));
  const int y = gsr_max_i(__float_as_int(fabsf(c)), __float_as_int(fabsf(d)));
  return __int_as_float(wave_max_i(gsr_max_i(x, y)));
}

__device__ __forceinline__ void unit_of(float most, float top, float* unit, float* inv) {
  const bool none = most < kUnitTiny;
  *unit = none ? 0.f : most * (1.f / top);
  *inv = none ? 0.f : 1.f / *unit;
}

__device__ __forceinline__ int adam_tensor(const AdamList& list, uint32_t block) {
  int lo = 0, hi = list.count - 1;
  while (lo < hi) {   // the last tensor whose first workgroup is not past this one
    const int mid = (lo + hi + 1) / 2;
    if (list.first[mid] <= block) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// UNBIASED: how moments of 8 bits are rounded.
template <typename P, typename G, int BITS, bool UNBIASED>
__global__ __launch_bounds__(256) void k_adamw(AdamList list, gsr_adamw_args a, AdamScalars host) {
  const int k = adam_tensor(list, blockIdx.x);
  const gsr_adamw_tensor& t = list.t[k];
  const AdamScalars s =
      t.step || a.lr_dev ? adam_scalars(a, a.lr_dev ? (double)*a.lr_dev : a.lr, t.step ? *t.step : a.step) : host;
  const int64_t begin = (int64_t)(blockIdx.x - list.first[k]) * kAdamChunk;
  P* p = (P*)t.p;
  const G* g = (const G*)t.g;
  const int lane = threadIdx.x % 64;
#pragma unroll
  for (int j = 0; j < kAdamChunk / 1024; ++j) {
    const int64_t blk = begin / kAdamBlock + j * 4 + threadIdx.x / 64;   // this wave's 256 elements
    const int64_t at = blk * kAdamBlock + lane * 4, n = t.n - at;
    if (blk * kAdamBlock >= t.n) break;   // the whole wave: the reductions below keep every lane
    float pv[4], gv[4], m[4], v[4], root[4];
    load_upto(p + at, n, pv);
    load_upto(g + at, n, gv);
    if constexpr (BITS == 32) {
      load_upto((const float*)t.m + at, n, m);
      load_upto((const float*)t.v + at, n, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) adam_element(s, gv[i], pv[i], m[i], v[i], root[i]);
      store_upto((float*)t.m + at, n, m);
      store_upto((float*)t.v + at, n, v);
    } else {
      uint8_t *mc = (uint8_t*)t.m + at, *vc = (uint8_t*)t.v + at;
      uint32_t mw = 0, vw = 0;
      if (n >= 4) {
        __builtin_memcpy(&mw, mc, 4);
        __builtin_memcpy(&vw, vc, 4);
      } else {
        for (int i = 0; i < n; ++i) {
          mw |= (uint32_t)mc[i] << (8 * i);
          vw |= (uint32_t)vc[i] << (8 * i);
        }
      }
      const float mu = t.m_unit[blk], vu = t.v_unit[blk];
      m[0] = __builtin_amdgcn_cvt_f32_fp8(mw, 0) * mu;
      m[1] = __builtin_amdgcn_cvt_f32_fp8(mw, 1) * mu;
      m[2] = __builtin_amdgcn_cvt_f32_fp8(mw, 2) * mu;
      m[3] = __builtin_amdgcn_cvt_f32_fp8(mw, 3) * mu;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float r = root_value((vw >> (8 * i)) & 255u, vu);
        v[i] = r * r;
        adam_element(s, gv[i], pv[i], m[i], v[i], root[i]);
        if (i >= n) m[i] = root[i] = 0.f;   // past the tensor's end
      }
      float nmu, minv, nvu, vinv;
      unit_of(wave_max_abs(m[0], m[1], m[2], m[3]), kMeanTop, &nmu, &minv);
      unit_of(wave_max_abs(root[0], root[1], root[2], root[3]), kRootTop, &nvu, &vinv);
      if (lane == 0) {
        t.m_unit[blk] = nmu;
        t.v_unit[blk] = nvu;
      }
      float q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // (a product a rounding above the top stays the top; NaN stays NaN)
        q[i] = m[i] * minv;
        q[i] = q[i] > kMeanTop ? kMeanTop : q[i] < -kMeanTop ? -kMeanTop : q[i];
      }
      uint32_t draw[4];
      if constexpr (UNBIASED) {
        const uint64_t count = (uint64_t)(t.step ? *t.step : a.step);
        const uint32_t block = (uint32_t)blk + (k == 0 ? list.skip * (kAdamChunk / kAdamBlock) : 0u);   // of the tensor
        const uint32_t base = mixed(mixed((uint32_t)count + mixed((uint32_t)(count >> 32))) + block);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          draw[i] = mixed(base ^ (uint32_t)(lane * 4 + i));
          q[i] = mean_unbiased(q[i], draw[i]);
          draw[i] = (draw[i] ^ draw[i] >> 15) * 0x9E3779B9u;   // the root's
        }
      }
      mw = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      mw = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], mw, true);
      vw = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t c = UNBIASED ? root_unbiased(root[i] * vinv, draw[i]) : root_code(root[i] * vinv);
        if (c == 0 && root[i] > 0.f && nvu != 0.f) c = 1;
        vw |= c << (8 * i);
      }
      if (n >= 4) {
        __builtin_memcpy(mc, &mw, 4);
        __builtin_memcpy(vc, &vw, 4);
      } else {
        for (int i = 0; i < n; ++i) {
          mc[i] = (uint8_t)(mw >> (8 * i));
          vc[i] = (uint8_t)(vw >> (8 * i));
        }
      }
    }
    store_upto(p + at, n, pv);
  }
}

// The roots that 8-bit codes stand for: four a lane, 5 bytes an element.
__global__ __launch_bounds__(256) void k_decode_root(const uint8_t* code, const float* unit, int64_t n, float* out) {
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; at < n; at += (int64_t)gridDim.x * 1024) {
    const float u = unit[at / kAdamBlock];
    float v[4];
    uint32_t w = 0;
    if (n - at >= 4) {
      __builtin_memcpy(&w, code + at, 4);
    } else {
      for (int i = 0; i < n - at; ++i) w |= (uint32_t)code[at + i] << (8 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = root_value((w >> (8 * i)) & 255u, u);
    store_upto(out + at, n - at, v);
  }
}

template <typename P, typename G>
static void adamw_launch(const AdamList& list, const gsr_adamw_args& a, const AdamScalars& s, hipStream_t st) {
  if (a.bits == 32) {
    k_adamw<P, G, 32, false><<<list.first[list.count], 256, 0, st>>>(list, a, s);
  } else if (a.rounding == GSR_ROUND_NEAREST) {
    k_adamw<P, G, 8, false><<<list.first[list.count], 256, 0, st>>>(list, a, s);
  } else {
    k_adamw<P, G, 8, true><<<list.first[list.count], 256, 0, st>>>(list, a, s);
  }
}

template <typename P>
static void adamw_launch(int gtype, const AdamList& list, const gsr_adamw_args& a, const AdamScalars& s, hipStream_t st) {
  if (gtype == GSR_F32) {
    adamw_launch<P, float>(list, a, s, st);
  } else if (gtype == GSR_BF16) {
    adamw_launch<P, bf16>(list, a, s, st);
  } else {
    adamw_launch<P, f16>(list, a, s, st);
  }
}

}  // namespace gsr

using namespace gsr;

extern "C" int gsr_adamw_step(const gsr_adamw_tensor* tensors, int32_t count, int32_t ptype, int32_t gtype,
                              const gsr_adamw_args* args, void* stream) {
  GSR_REQUIRE(args && (tensors || count == 0) && count >= 0, "gsr_adamw_step: bad list (count %d)", count);
  const gsr_adamw_args& a = *args;
  GSR_REQUIRE(known_type(ptype) && known_type(gtype), "gsr_adamw_step: bad type (%d, %d)", ptype, gtype);
  GSR_REQUIRE(a.bits == 32 || a.bits == 8, "gsr_adamw_step: moments in 32 or 8 bits, not %d", a.bits);
  GSR_REQUIRE(a.rounding == GSR_ROUND_NEAREST || a.rounding == GSR_ROUND_UNBIASED, "gsr_adamw_step: bad rounding %d", a.rounding);
  GSR_REQUIRE(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0, "gsr_adamw_step: bad betas (%g, %g)",
              a.beta1, a.beta2);
  GSR_REQUIRE(a.eps >= 0.0 && a.weight_decay >= 0.0 && (a.lr_dev || a.lr >= 0.0), "gsr_adamw_step: bad lr, eps or weight decay");
  for (int i = 0; i < count; ++i) {
    const gsr_adamw_tensor& t = tensors[i];
    GSR_REQUIRE(t.n >= 0 && t.n <= (int64_t)1 << 40, "gsr_adamw_step: tensor %d: bad length %lld", i, (long long)t.n);
    GSR_REQUIRE(t.n == 0 || (t.p && t.g && t.m && t.v && (a.bits == 32 || (t.m_unit && t.v_unit))),
                "gsr_adamw_step: tensor %d: null pointer", i);
    GSR_REQUIRE(t.step || a.step >= 1, "gsr_adamw_step: bad step %lld (the first is 1)", (long long)a.step);
  }
  const AdamScalars s = a.lr_dev || a.step < 1 ? AdamScalars{} : adam_scalars(a, a.lr, a.step);
  const auto st = (hipStream_t)stream;
  const uint32_t most = 1u << 23;   // workgroups a launch: below 2^32 threads
  AdamList list;
  list.count = 0;
  list.skip = 0;
  list.first[0] = 0;
  const auto flush = [&]() {
    if (list.count == 0) return;
    if (ptype == GSR_F32) {
      adamw_launch<float>(gtype, list, a, s, st);
    } else if (ptype == GSR_BF16) {
      adamw_launch<bf16>(gtype, list, a, s, st);
    } else {
      adamw_launch<f16>(gtype, list, a, s, st);
    }
    list.count = 0;
  };
  for (int i = 0; i < count; ++i) {
    gsr_adamw_tensor t = tensors[i];
    uint32_t taken = 0;   // workgroups
    while (t.n > 0) {   // a tensor that does not fit what is left of a launch is cut at a workgroup's border
      const uint32_t used = list.first[list.count];
      int64_t n = t.n < (int64_t)(most - used) * kAdamChunk ? t.n : (int64_t)(most - used) * kAdamChunk;
      if (list.count == 0) list.skip = taken;   // (a cut tensor goes on as the next launch's first)
      list.t[list.count] = t;
      list.t[list.count].n = n;
      list.first[++list.count] = used + (uint32_t)ceil_div64(n, kAdamChunk);
      taken += (uint32_t)ceil_div64(n, kAdamChunk);
      t.n -= n;
      t.p = (char*)t.p + n * (int64_t)type_size(ptype);
      t.g = (const char*)t.g + n * (int64_t)type_size(gtype);
      t.m = (char*)t.m + n * (a.bits / 8);
      t.v = (char*)t.v + n * (a.bits / 8);
      if (a.bits == 8) {
        t.m_unit += n / kAdamBlock;
        t.v_unit += n / kAdamBlock;
      }
      if (list.count == kAdamTensors || list.first[list.count] == most) flush();
    }
  }
  flush();
  GSR_LAUNCH_CHECK("gsr_adamw_step");
  return 0;
}

extern "C" int gsr_adamw_decode_root(const uint8_t* codes, const float* units, int64_t n, float* out, void* stream) {
  GSR_REQUIRE(n >= 0, "gsr_adamw_decode_root: bad n %lld", (long long)n);
  if (n == 0) return 0;
  GSR_REQUIRE(codes && units && out, "gsr_adamw_decode_root: null pointer");
  const int64_t blocks = ceil_div64(n, 1024);
  k_decode_root<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, (hipStream_t)stream>>>(codes, units, n, out);
  GSR_LAUNCH_CHECK("gsr_adamw_decode_root");
  return 0;
}
