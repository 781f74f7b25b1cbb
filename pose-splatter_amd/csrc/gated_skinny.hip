// The gated block's projections of few rows (up to 64), where reading the weights is all there is.
//
// A workgroup owns 16 columns of g and of u and all rows.  Its waves take the K steps in turn, so
// that neighbouring waves read neighbouring lines; each lane loads its 16 bytes of a weight row
// straight into the matrix instruction's operand (lane % 16 the row, lane / 16 the K group), four
// steps at a time to keep loads in flight.  The waves' sums meet in shared memory, are added in
// order, and the activation follows there: no partial results in memory, one launch.  1 x 4096 ->
// 11264 bf16: 35 us, 5.3 TB/s of weights.
#include "gated_skinny.h"

namespace gsr {

typedef float sk_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 sk_v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 sk_v8h __attribute__((ext_vector_type(8)));

// 16 bytes of T as the matrix instruction takes them.
template <typename T>
struct Chunk {
  static constexpr int V = 16 / sizeof(T);
  Pack<T, V> v;
  __device__ __forceinline__ void load(const T* p) { v = *(const Pack<T, V>*)p; }
  __device__ __forceinline__ void load_part(const T* p, int64_t n) {   // the first n elements, then zeros
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = i < n ? p[i] : from_f<T>(0.f);
  }
};

__device__ __forceinline__ sk_v4f skinny_mma(const Chunk<bf16>& a, const Chunk<bf16>& b, sk_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sk_v8bf, a.v), __builtin_bit_cast(sk_v8bf, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ sk_v4f skinny_mma(const Chunk<f16>& a, const Chunk<f16>& b, sk_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sk_v8h, a.v), __builtin_bit_cast(sk_v8h, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ sk_v4f skinny_mma(const Chunk<float>& a, const Chunk<float>& b, sk_v4f c) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v.v[s], b.v.v[s], c, 0, 0, 0);
  return c;
}

// MT: blocks of 16 rows.  GRAD: dgu and parts [2][hidden] (the column sums, or NULL) in the place of h.
template <typename T, int MT, int WAVES, bool GRAD>
__global__ __launch_bounds__(WAVES * 64) void k_skinny(GatedSkinny a) {
  constexpr int V = Chunk<T>::V, KS = 4 * V, STEPS = 4;
  __shared__ float lds[WAVES][2][MT][256];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const GatedShape s = a.s;
  const int64_t n0 = (int64_t)blockIdx.x * 16, k_lane = lane / 16 * V;
  // rows past the last read the last one again: their sums belong to no output
  const int64_t wn = n0 + lane % 16 < s.hidden ? n0 + lane % 16 : s.hidden - 1;
  const T *wg = (const T*)a.wg + wn * s.dim + k_lane, *wu = (const T*)a.wu + wn * s.dim + k_lane;
  const T* x[MT];
  sk_v4f g[MT], u[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t r = m * 16 + lane % 16;
    x[m] = (const T*)a.x + (r < s.rows ? r : s.rows - 1) * a.x_stride + k_lane;
    g[m] = u[m] = sk_v4f{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t whole = s.dim / KS * KS;
  int64_t k = (int64_t)wave * KS;
  for (; k + (STEPS - 1) * WAVES * KS < whole; k += STEPS * WAVES * KS) {
    Chunk<T> cg[STEPS], cu[STEPS], cx[STEPS][MT];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int64_t at = k + j * WAVES * KS;
      cg[j].load(wg + at);
      cu[j].load(wu + at);
#pragma unroll
      for (int m = 0; m < MT; ++m) cx[j][m].load(x[m] + at);
    }
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        g[m] = skinny_mma(cg[j], cx[j][m], g[m]);
        u[m] = skinny_mma(cu[j], cx[j][m], u[m]);
      }
  }
  for (; k < s.dim; k += WAVES * KS) {
    Chunk<T> cg, cu, cx[MT];
    const int64_t n = s.dim - k - k_lane;
    if (k < whole) {
      cg.load(wg + k);
      cu.load(wu + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) cx[m].load(x[m] + k);
    } else {
      cg.load_part(wg + k, n);
      cu.load_part(wu + k, n);
#pragma unroll
      for (int m = 0; m < MT; ++m) cx[m].load_part(x[m] + k, n);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      g[m] = skinny_mma(cg, cx[m], g[m]);
      u[m] = skinny_mma(cu, cx[m], u[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    *(sk_v4f*)&lds[wave][0][m][lane * 4] = g[m];
    *(sk_v4f*)&lds[wave][1][m][lane * 4] = u[m];
  }
  __syncthreads();
  const int64_t pad = gated_pad(s.hidden);
  for (int at = threadIdx.x; at < MT * 256; at += WAVES * 64) {
    const int mt = at / 256, m = at % 256 / 16, c = at % 16, from = (m + c / 4 * 16) * 4 + c % 4;
    const int64_t row = mt * 16 + m, n = n0 + c;
    const bool in = row < s.rows && n < s.hidden;
    float gv = 0.f, uv = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      gv += lds[w][0][mt][from];
      uv += lds[w][1][mt][from];
    }
    if (in && a.bg) {
      gv += to_f(((const T*)a.bg)[n]);
      uv += to_f(((const T*)a.bu)[n]);
    }
    const float one[1] = {gv};
    float act[1], slope[1];
    activate<T>(a.act, one, act, slope);
    if constexpr (!GRAD) {
      if (in) {
        if (a.kept) Kept<T>(a.kept, s.rows, s.hidden).store_one(row * pad + n, gv, uv);
        ((T*)a.h)[row * s.hidden + n] = from_f<T>(act[0] * uv);
      }
    } else {
      const float d = in ? to_f(((const T*)a.dh)[row * a.dh_stride + n]) : 0.f;
      gv = in ? d * uv * slope[0] : 0.f;   // (the padding holds zeros)
      uv = in ? d * act[0] : 0.f;
      if (row < s.rows) {
        const int64_t to = row * 2 * pad + n;
        if (a.dgu32) {
          ((float*)a.dgu)[to] = gv;
          ((float*)a.dgu)[to + pad] = uv;
        } else {
          ((T*)a.dgu)[to] = from_f<T>(gv);
          ((T*)a.dgu)[to + pad] = from_f<T>(uv);
        }
      }
      lds[0][0][mt][from] = gv;   // (this thread alone reads and writes the place)
      lds[0][1][mt][from] = uv;
    }
  }
  if (GRAD && a.parts) {
    __syncthreads();
    if (threadIdx.x < 32) {
      const int c = threadIdx.x % 16, which = threadIdx.x / 16;
      float v = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        for (int m = 0; m < 16; ++m) v += lds[0][which][mt][(m + c / 4 * 16) * 4 + c % 4];
      if (n0 + c < s.hidden) a.parts[which * s.hidden + n0 + c] = v;
    }
  }
}

template <typename T, int MT>
static void skinny_launch(const GatedSkinny& a, hipStream_t st) {
  // a workgroup's 16 columns are all its own: with fewer workgroups than CUs each takes 16 waves
  const int64_t blocks = (a.h ? ceil_div64(a.s.hidden, 16) : gated_pad(a.s.hidden) / 16);
  const bool few = blocks < 256;
  const unsigned grid = (unsigned)blocks;
  if (a.h && few) {
    k_skinny<T, MT, 16, false><<<grid, 1024, 0, st>>>(a);
  } else if (a.h) {
    k_skinny<T, MT, 8, false><<<grid, 512, 0, st>>>(a);
  } else if (few) {
    k_skinny<T, MT, 16, true><<<grid, 1024, 0, st>>>(a);
  } else {
    k_skinny<T, MT, 8, true><<<grid, 512, 0, st>>>(a);
  }
}

template <typename T>
static void skinny_rows(const GatedSkinny& a, hipStream_t st) {
  if (a.s.rows <= 16) {
    skinny_launch<T, 1>(a, st);
  } else if (a.s.rows <= 32) {
    skinny_launch<T, 2>(a, st);
  } else {
    skinny_launch<T, 4>(a, st);
  }
}

void gated_skinny(int type, const GatedSkinny& a, hipStream_t st) {
  if (type == GSR_F32) {
    skinny_rows<float>(a, st);
  } else if (type == GSR_BF16) {
    skinny_rows<bf16>(a, st);
  } else {
    skinny_rows<f16>(a, st);
  }
}

}  // namespace gsr
