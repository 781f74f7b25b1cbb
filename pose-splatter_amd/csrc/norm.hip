// Layer norm over rows, forward and backward.
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (w dy - mean(w dy) - xhat mean(w dy xhat)),  dw = sum_rows dy xhat,  db = sum_rows dy
//
// Both passes are bound by memory: a row is read once and stays in registers while its mean,
// then its variance about that mean (two sums, so no cancellation of E[x^2] - mean^2) are
// reduced.  LANES lanes share a row -- part of a wave for short rows, a wave, or a whole
// workgroup -- each holding NV vectors of V elements.  Workgroups walk rows with the grid's stride,
// keep the weights (and the backward's dw and db) of their columns in registers and load the next
// row while they reduce this one.  Each backward workgroup writes one row of partial dw and db,
// which a second kernel adds in a fixed order: no atomics, the same bits every run.
// Sums, statistics and partials are fp32; only y, dx, dw and db are rounded to their types.
// 32768 x 4096 bf16: forward 104 us (5.2 TB/s), backward 159 (5.1 TB/s).
#include <type_traits>

#include "types.h"

namespace gsr {

// Workgroups of a backward at most, one partial row of dw and db each: those that run at once, three a
// CU with up to two vectors a lane, two with four (32768 x 4096 bf16: 161 us at 768, 194 at 512, 191 at
// 1024 where registers spill; 16384 x 8192: 171 at 512, 200 at 768).
constexpr int norm_most_parts(int nv) { return nv <= 2 ? 768 : 512; }
constexpr int kNormGrid = 2048;   // workgroups of a forward: up to eight a CU

template <typename T>
struct NormVec {
  static constexpr int V = sizeof(T) == 4 ? 4 : 8;   // 16 bytes
};

// Sum over the LANES lanes of a row, in all of them.  Workgroup rows (LANES > 64) go through
// `lds`, of which a caller alternates two halves so that one barrier a sum is enough.
template <int LANES, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds) {
  if constexpr (LANES < 64) {
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], d);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (LANES > 64) {
      constexpr int W = LANES / 64;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[i * W + threadIdx.x / 64] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += lds[i * W + w];
        v[i] = s;
      }
    }
  }
}

// The columns of a lane's k-th vector of a row.  EARLY, for rows of a vector or more: where one does not end
// on a whole vector, its last one ends with the row instead and begins skip() columns early.  Those
// belong to the lane before too, which writes the same values to them; sums leave them out.  Without
// it that lane goes element by element, and every row's wave waits for up to seven more loads and
// stores: 32768 x 4095 bf16 forward 166 us against 121, backward 261 against 193.
template <int V, int LANES, bool EARLY>
struct NormCols {
  using Index = std::conditional_t<EARLY, int, int64_t>;   // (64 bits: what the backward without it schedules best)
  Index dim;
  int lane, last, early;   // the vector that ends the row (of some lane), and how early it begins
  __device__ __forceinline__ NormCols(int64_t d) : dim((Index)d), lane(threadIdx.x % LANES), last(((int)d - 1) / (LANES * V)) {
    const int c = (last * LANES + lane) * V;
    early = EARLY && c < dim && c + V > dim ? c + V - (int)dim : 0;
  }
  // Makes what follows compute from `early` anew: kept over the rows, it would take registers by the dozen.
  __device__ __forceinline__ void forget() {
    if constexpr (EARLY) asm volatile("" : "+v"(early));
  }
  __device__ __forceinline__ int skip(int k) const { return EARLY && k == last ? early : 0; }
  __device__ __forceinline__ Index at(int k) const { return (Index)(k * LANES + lane) * V - skip(k); }
  __device__ __forceinline__ Index n(int k) const {
    const Index left = dim - (Index)(k * LANES + lane) * V;
    return EARLY ? (left > 0 ? V : 0) : left;
  }
  __device__ __forceinline__ bool in(int k, int i) const { return i >= skip(k) && i < n(k); }
};

template <typename T, int LANES, int NV, bool EARLY>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void k_norm_fwd(const T* x, int64_t rows, int64_t dim, int64_t stride,
                                                                        const void* w, const void* b, int wtype, float eps,
                                                                        T* y, float2* stats) {
  constexpr int V = NormVec<T>::V, THREADS = LANES > 256 ? LANES : 256, RPB = THREADS / LANES;
  constexpr bool HOLD = LANES <= 256;   // (1024 threads leave no registers for the weights)
  __shared__ float lds[LANES > 64 ? 2 * (LANES / 64) : 1];
  const int lane = threadIdx.x % LANES;
  NormCols<V, LANES, EARLY> cols(dim);
  float wv[HOLD ? NV : 1][V], bv[HOLD ? NV : 1][V];
  if constexpr (HOLD)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      load_param(w, wtype, cols.at(k), cols.n(k), wv[k], 1.f);
      load_param(b, wtype, cols.at(k), cols.n(k), bv[k], 0.f);
    }
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  Raw<T> next[NV];
  const auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      next[k].load(x + r * stride + cols.at(k), cols.n(k));
    }
  };
  if (row < rows) fetch(row);
  for (; row < rows; row += step) {
    float v[NV][V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] = next[k].at(i);
        s[0] += !EARLY || i >= cols.skip(k) ? v[k][i] : 0.f;   // (columns that are not there hold zeros)
      }
    if (row + step < rows) fetch(row + step);
    cols.forget();
    row_sum<LANES>(s, lds);
    const float mean = s[0] / (float)dim;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] -= mean;
        s[0] += cols.in(k, i) ? v[k][i] * v[k][i] : 0.f;
      }
    }
    row_sum<LANES>(s, lds + (LANES > 64 ? LANES / 64 : 0));
    const float rstd = 1.f / sqrtf(s[0] / (float)dim + eps);
    if (stats && lane == 0) stats[row] = make_float2(mean, rstd);
    T* yr = y + row * dim;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (cols.n(k) > 0) {
        const int h = HOLD ? k : 0;
        if constexpr (!HOLD) {
          load_param(w, wtype, cols.at(k), cols.n(k), wv[0], 1.f);
          load_param(b, wtype, cols.at(k), cols.n(k), bv[0], 0.f);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = v[k][i] * rstd * wv[h][i] + bv[h][i];
        store_upto(yr + cols.at(k), cols.n(k), v[k]);
      }
    }
  }
}

// Rows of any length: the row is read three times (from cache after the first).
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(const T* x, int64_t rows, int64_t dim, int64_t stride, const void* w,
                                                        const void* b, int wtype, float eps, T* y, float2* stats) {
  constexpr int V = NormVec<T>::V;
  __shared__ float lds[2 * 16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * stride;
    float s[1] = {0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < dim; c += 1024 * V) {
      float v[V];
      load_upto(xr + c, dim - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += v[i];
    }
    row_sum<1024>(s, lds);
    const float mean = s[0] / (float)dim;
    s[0] = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < dim; c += 1024 * V) {
      float v[V];
      load_upto(xr + c, dim - c, v, mean);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += (v[i] - mean) * (v[i] - mean);
    }
    row_sum<1024>(s, lds + 16);
    const float rstd = 1.f / sqrtf(s[0] / (float)dim + eps);
    if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
    for (int64_t c = (int64_t)threadIdx.x * V; c < dim; c += 1024 * V) {
      float v[V], wv[V], bv[V];
      load_upto(xr + c, dim - c, v);
      load_param(w, wtype, c, dim - c, wv, 1.f);
      load_param(b, wtype, c, dim - c, bv, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - mean) * rstd * wv[i] + bv[i];
      store_upto(y + row * dim + c, dim - c, v);
    }
  }
}

// parts: [gridDim.x][2][dim] partial sums of dw and db (NULL: neither is wanted).  x and dy stay as they
// were loaded (a row's two values of 16 bits in one register) and are widened again for dx: the
// registers saved are waves that keep more loads in flight.
template <typename T, int LANES, int NV, bool EARLY>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256, LANES > 256 ? 1 : NV <= 2 ? 3 : 2) void k_norm_bwd(
    const T* x, const T* dy, int64_t rows, int64_t dim, int64_t stride, int64_t dy_stride, const void* w, int wtype,
    const float2* stats, T* dx, float* parts) {
  constexpr int V = NormVec<T>::V, THREADS = LANES > 256 ? LANES : 256, RPB = THREADS / LANES;
  constexpr int W = LANES / 64;
  constexpr bool HOLD = LANES <= 256;   // weights and the next row in registers (1024 threads have none left)
  __shared__ float lds[LANES > 64 ? 4 * W : 1];
  const float inv = 1.f / (float)dim;
  NormCols<V, LANES, EARLY> cols(dim);
  float wv[HOLD ? NV : 1][V], aw[NV][V] = {}, ab[NV][V] = {};
  const auto weights = [&](int k) {
    load_param(w, wtype, cols.at(k), cols.n(k), wv[HOLD ? k : 0], 1.f);
  };
  if constexpr (HOLD)
#pragma unroll
    for (int k = 0; k < NV; ++k) weights(k);
  int half = 0;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  Raw<T> nx[NV], ng[NV];
  float2 next_st;
  const auto fetch = [&](int64_t r) {
    next_st = stats[r];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      nx[k].load(x + r * stride + cols.at(k), cols.n(k));
      ng[k].load(dy + r * dy_stride + cols.at(k), cols.n(k));
    }
  };
  if (HOLD && row < rows) fetch(row);
  for (; row < rows; row += step) {
    if constexpr (!HOLD) fetch(row);
    const float2 st = next_st;
    Raw<T> cx[NV], cg[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) cx[k] = nx[k], cg[k] = ng[k];
    if (HOLD && row + step < rows) fetch(row + step);
    cols.forget();
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (!HOLD) weights(k);
      const int skip = cols.skip(k);   // (columns that are not there hold zeros of dy)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = (cx[k].at(i) - st.x) * st.y, d = !EARLY || i >= skip ? cg[k].at(i) : 0.f;
        aw[k][i] += d * z;
        ab[k][i] += d;
        s[0] += d * wv[HOLD ? k : 0][i];
        s[1] += d * wv[HOLD ? k : 0][i] * z;
      }
    }
    row_sum<LANES>(s, lds + half * 2 * W);
    half ^= 1;
    if (dx) {
      const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if constexpr (!HOLD) weights(k);
        float g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float z = (cx[k].at(i) - st.x) * st.y;
          g[i] = (cg[k].at(i) * wv[HOLD ? k : 0][i] - m0 - z * m1) * st.y;
        }
        if (cols.n(k) > 0) store_upto(dx + row * dim + cols.at(k), cols.n(k), g);
      }
    }
  }
  if (!parts) return;
  // the workgroup's rows: lanes of a wave that hold the same columns, then the waves through LDS
  float* out = parts + (int64_t)blockIdx.x * 2 * dim;
  if constexpr (LANES < 64) {
#pragma unroll
    for (int d = LANES; d < 64; d <<= 1)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          aw[k][i] += __shfl_xor(aw[k][i], d);
          ab[k][i] += __shfl_xor(ab[k][i], d);
        }
  }
  if constexpr (LANES <= 64) {
    constexpr int COLS = LANES * V;
    __shared__ float sum[4][2][COLS];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (threadIdx.x % 64 < LANES)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (!EARLY || cols.in(k, i)) {   // (from the vector's own first column on: inside these COLS)
            const int at = (int)cols.at(k) + i - k * COLS;
            sum[threadIdx.x / 64][0][at] = aw[k][i];
            sum[threadIdx.x / 64][1][at] = ab[k][i];
          }
      __syncthreads();
      for (int j = threadIdx.x; j < 2 * COLS; j += THREADS) {
        const int which = j / COLS, c = j % COLS;
        const int64_t col = (int64_t)k * COLS + c;
        if (col < dim)
          out[which * dim + col] = (sum[0][which][c] + sum[1][which][c]) + (sum[2][which][c] + sum[3][which][c]);
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (EARLY && cols.skip(k) > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (cols.in(k, i)) out[cols.at(k) + i] = aw[k][i], out[dim + cols.at(k) + i] = ab[k][i];
      } else if (cols.n(k) > 0) {
        store_upto(out + cols.at(k), cols.n(k), aw[k]);
        store_upto(out + dim + cols.at(k), cols.n(k), ab[k]);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(const T* x, const T* dy, int64_t rows, int64_t dim, int64_t stride,
                                                        int64_t dy_stride, const void* w, int wtype, const float2* stats,
                                                        T* dx) {
  constexpr int V = NormVec<T>::V;
  __shared__ float lds[2][2 * 16];
  int half = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, half ^= 1) {
    const float2 st = stats[row];
    const T *xr = x + row * stride, *gr = dy + row * dy_stride;
    float s[2] = {0.f, 0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < dim; c += 1024 * V) {
      float v[V], g[V], wv[V];
      load_upto(xr + c, dim - c, v, st.x);
      load_upto(gr + c, dim - c, g);
      load_param(w, wtype, c, dim - c, wv, 1.f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[0] += g[i] * wv[i];
        s[1] += g[i] * wv[i] * ((v[i] - st.x) * st.y);
      }
    }
    row_sum<1024>(s, lds[half]);
    const float m0 = s[0] / (float)dim, m1 = s[1] / (float)dim;
    for (int64_t c = (int64_t)threadIdx.x * V; c < dim; c += 1024 * V) {
      float v[V], g[V], wv[V];
      load_upto(xr + c, dim - c, v, st.x);
      load_upto(gr + c, dim - c, g);
      load_param(w, wtype, c, dim - c, wv, 1.f);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = (g[i] * wv[i] - m0 - (v[i] - st.x) * st.y * m1) * st.y;
      store_upto(dx + row * dim + c, dim - c, g);
    }
  }
}

// Partial dw/db of long rows: a thread per column, blockIdx.y's share of the rows.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_cols(const T* x, const T* dy, int64_t rows, int64_t dim, int64_t stride,
                                                   int64_t dy_stride, const float2* stats, float* parts) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= dim) return;
  float aw = 0.f, ab = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float2 st = stats[row];
    const float g = to_f(dy[row * dy_stride + c]);
    aw += g * ((to_f(x[row * stride + c]) - st.x) * st.y);
    ab += g;
  }
  parts[(int64_t)blockIdx.y * 2 * dim + c] = aw;
  parts[(int64_t)blockIdx.y * 2 * dim + dim + c] = ab;
}

// dw, db = the sum of n partial rows: 16 groups of lanes a column, each a fixed share of the
// rows, then the groups in order.  Workgroups walk the columns with the grid's stride.
__global__ __launch_bounds__(1024) void k_norm_join(const float* parts, int n, int64_t dim, void* dw, void* db, int wtype) {
  __shared__ float sum[16][65];
  const int col = threadIdx.x % 64, grp = threadIdx.x / 64;
  for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < 2 * dim; c0 += (int64_t)gridDim.x * 64) {
    const int64_t c = c0 + col;
    float s = 0.f;
    if (c < 2 * dim) {
#pragma unroll 8
      for (int r = grp; r < n; r += 16) s += parts[(int64_t)r * 2 * dim + c];
    }
    sum[grp][col] = s;
    __syncthreads();
    if (grp == 0 && c < 2 * dim) {
#pragma unroll
      for (int k = 1; k < 16; ++k) s += sum[k][col];
      if (c < dim) {
        if (dw) store_param(dw, wtype, c, s);
      } else if (db) {
        store_param(db, wtype, c - dim, s);
      }
    }
    __syncthreads();
  }
}

// Vectors a row -> the layout that holds it: lanes a row (a power of two up to a wave, then 256
// and 1024) and vectors a lane; 0 lanes: longer than registers hold.
static void norm_layout(int64_t vecs, int* lanes, int* nv) {
  int l = 1;
  while (l < 64 && l < vecs) l <<= 1;
  *lanes = l;
  *nv = 1;
  if (vecs <= 64) return;
  if (vecs <= 256) {
    *nv = vecs <= 128 ? 2 : 4;
  } else if (vecs <= 1024) {
    *lanes = 256;
    *nv = vecs <= 512 ? 2 : 4;
  } else if (vecs <= 4096) {
    *lanes = 1024;
    *nv = vecs <= 2048 ? 2 : 4;
  } else {
    *lanes = 0;
  }
}

static unsigned norm_grid(int64_t blocks) { return (unsigned)(blocks < kNormGrid ? blocks : kNormGrid); }

#define GSR_NORM_DISPATCH(CALL)                 \
  switch (lanes * 8 + nv) {                     \
    case 1 * 8 + 1: CALL(1, 1); break;          \
    case 2 * 8 + 1: CALL(2, 1); break;          \
    case 4 * 8 + 1: CALL(4, 1); break;          \
    case 8 * 8 + 1: CALL(8, 1); break;          \
    case 16 * 8 + 1: CALL(16, 1); break;        \
    case 32 * 8 + 1: CALL(32, 1); break;        \
    case 64 * 8 + 1: CALL(64, 1); break;        \
    case 64 * 8 + 2: CALL(64, 2); break;        \
    case 64 * 8 + 4: CALL(64, 4); break;        \
    case 256 * 8 + 2: CALL(256, 2); break;      \
    case 256 * 8 + 4: CALL(256, 4); break;      \
    case 1024 * 8 + 2: CALL(1024, 2); break;    \
    case 1024 * 8 + 4: CALL(1024, 4); break;    \
  }

// Partial rows of dw/db that a backward writes.
static int norm_parts(int64_t rows, int64_t dim, int xtype) {
  int lanes, nv;
  norm_layout(ceil_div64(dim, xtype == GSR_F32 ? 4 : 8), &lanes, &nv);
  const int rpb = lanes == 0 || lanes > 256 ? 1 : 256 / lanes;
  const int64_t blocks = ceil_div64(rows, rpb);
  // enough rows a part that writing and joining it stays small beside reading them, but a part a CU
  int64_t most = lanes == 0 ? 64 : blocks / 8 < 256 ? 256 : blocks / 8;
  if (lanes && most > norm_most_parts(nv)) most = norm_most_parts(nv);
  return (int)(blocks < most ? blocks : most);
}

template <typename T>
static void norm_fwd(const void* x, int64_t rows, int64_t dim, int64_t stride, const void* w, const void* b, int wtype,
                     float eps, void* y, float* stats, hipStream_t s) {
  int lanes, nv;
  norm_layout(ceil_div64(dim, NormVec<T>::V), &lanes, &nv);
  if (lanes == 0) {
    k_norm_fwd_long<T><<<norm_grid(rows), 1024, 0, s>>>((const T*)x, rows, dim, stride, w, b, wtype, eps, (T*)y, (float2*)stats);
    return;
  }
  const int rpb = lanes > 256 ? 1 : 256 / lanes;
  const unsigned grid = norm_grid(ceil_div64(rows, rpb));
  void (*f)(const T*, int64_t, int64_t, int64_t, const void*, const void*, int, float, T*, float2*) = nullptr;
#define GSR_CALL(L, N) f = dim >= NormVec<T>::V ? k_norm_fwd<T, L, N, true> : k_norm_fwd<T, L, N, false>
  GSR_NORM_DISPATCH(GSR_CALL)
#undef GSR_CALL
  f<<<grid, lanes > 256 ? lanes : 256, 0, s>>>((const T*)x, rows, dim, stride, w, b, wtype, eps, (T*)y, (float2*)stats);
}

template <typename T>
static void norm_bwd(const void* x, const void* dy, int64_t rows, int64_t dim, int64_t stride, int64_t dy_stride,
                     const void* w, int wtype, const float* stats, void* dx, float* parts, int n, hipStream_t s) {
  int lanes, nv;
  norm_layout(ceil_div64(dim, NormVec<T>::V), &lanes, &nv);
  if (lanes == 0) {
    if (dx)
      k_norm_bwd_long<T><<<norm_grid(rows), 1024, 0, s>>>((const T*)x, (const T*)dy, rows, dim, stride, dy_stride, w, wtype,
                                                         (const float2*)stats, (T*)dx);
    if (parts)
      k_norm_cols<T><<<dim3((unsigned)ceil_div64(dim, 256), n), 256, 0, s>>>((const T*)x, (const T*)dy, rows, dim, stride,
                                                                            dy_stride, (const float2*)stats, parts);
    return;
  }
  // (early vectors take registers that 32 values a lane, or 1024 lanes, do not leave: 8359 x 7187 bf16 123 us, 118 without)
  constexpr int V = NormVec<T>::V;
  void (*f)(const T*, const T*, int64_t, int64_t, int64_t, int64_t, const void*, int, const float2*, T*, float*) = nullptr;
#define GSR_CALL(L, N) f = dim >= V ? k_norm_bwd<T, L, N, ((N) * V < 32 && (L) <= 256)> : k_norm_bwd<T, L, N, false>
  GSR_NORM_DISPATCH(GSR_CALL)
#undef GSR_CALL
  f<<<n, lanes > 256 ? lanes : 256, 0, s>>>((const T*)x, (const T*)dy, rows, dim, stride, dy_stride, w, wtype, (const float2*)stats,
                                            (T*)dx, parts);
}

static int norm_check(const char* who, int64_t rows, int64_t dim, int64_t stride, int xtype, int wtype) {
  GSR_REQUIRE(rows >= 0 && rows <= INT32_MAX, "%s: bad rows %lld", who, (long long)rows);
  GSR_REQUIRE(dim >= 1 && dim <= INT32_MAX, "%s: bad dim %lld", who, (long long)dim);
  GSR_REQUIRE(rows <= 1 || stride >= dim, "%s: row stride %lld below dim %lld", who, (long long)stride, (long long)dim);
  GSR_REQUIRE(known_type(xtype) && known_type(wtype), "%s: bad type (%d, %d)", who, xtype, wtype);
  return 0;
}

}  // namespace gsr

using namespace gsr;

extern "C" int gsr_layer_norm_fwd(const void* x, int64_t rows, int64_t dim, int64_t stride, int32_t xtype, const void* w,
                                  const void* b, int32_t wtype, float eps, void* y, float* stats, void* stream) {
  if (const int e = norm_check("gsr_layer_norm_fwd", rows, dim, stride, xtype, wtype)) return e;
  GSR_REQUIRE(eps >= 0.f, "gsr_layer_norm_fwd: bad eps %g", eps);
  if (rows == 0) return 0;
  GSR_REQUIRE(x && y, "gsr_layer_norm_fwd: null x or y");
  const auto s = (hipStream_t)stream;
  if (xtype == GSR_F32) {
    norm_fwd<float>(x, rows, dim, stride, w, b, wtype, eps, y, stats, s);
  } else if (xtype == GSR_BF16) {
    norm_fwd<bf16>(x, rows, dim, stride, w, b, wtype, eps, y, stats, s);
  } else {
    norm_fwd<f16>(x, rows, dim, stride, w, b, wtype, eps, y, stats, s);
  }
  GSR_LAUNCH_CHECK("gsr_layer_norm_fwd");
  return 0;
}

extern "C" size_t gsr_layer_norm_workspace(int64_t rows, int64_t dim, int32_t xtype) {
  if (rows <= 0 || dim <= 0 || !known_type(xtype)) return 0;
  return (size_t)norm_parts(rows, dim, xtype) * 2 * (size_t)dim * sizeof(float);
}

extern "C" int gsr_layer_norm_bwd(const void* x, const void* dy, int64_t rows, int64_t dim, int64_t stride,
                                  int64_t dy_stride, int32_t xtype, const void* w, int32_t wtype, const float* stats,
                                  void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int e = norm_check("gsr_layer_norm_bwd", rows, dim, stride, xtype, wtype)) return e;
  GSR_REQUIRE(rows <= 1 || dy_stride >= dim, "gsr_layer_norm_bwd: dy row stride %lld below dim", (long long)dy_stride);
  const bool sums = dw || db;
  if (!dx && !sums) return 0;
  const auto s = (hipStream_t)stream;
  const int n = rows ? norm_parts(rows, dim, xtype) : 0;
  if (sums)
    GSR_REQUIRE(workspace_bytes >= gsr_layer_norm_workspace(rows, dim, xtype) && (workspace || !rows),
                "gsr_layer_norm_bwd: workspace too small (%zu bytes)", workspace_bytes);
  if (rows) {
    GSR_REQUIRE(x && dy && stats, "gsr_layer_norm_bwd: null x, dy or stats");
    float* parts = sums ? (float*)workspace : nullptr;
    if (xtype == GSR_F32) {
      norm_bwd<float>(x, dy, rows, dim, stride, dy_stride, w, wtype, stats, dx, parts, n, s);
    } else if (xtype == GSR_BF16) {
      norm_bwd<bf16>(x, dy, rows, dim, stride, dy_stride, w, wtype, stats, dx, parts, n, s);
    } else {
      norm_bwd<f16>(x, dy, rows, dim, stride, dy_stride, w, wtype, stats, dx, parts, n, s);
    }
    GSR_LAUNCH_CHECK("gsr_layer_norm_bwd");
  }
  if (sums) {
    const int64_t blocks = ceil_div64(2 * dim, 64);   // (a launch holds less than 2^32 threads)
    k_norm_join<<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 1024, 0, s>>>((const float*)workspace, n, dim, dw, db, wtype);
    GSR_LAUNCH_CHECK("gsr_layer_norm_bwd (join)");
  }
  return 0;
}
