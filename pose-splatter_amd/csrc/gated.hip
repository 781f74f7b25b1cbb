// Gated block  h = act(x Wg^T + bg) * (x Wu^T + bu)  and its backward pass.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg, dbu = column sums of dg, du
//
// Three products.  The forward's one launch computes both projections of a tile side by side, so
// that g, u and the activation never leave registers.  The backward needs g and u again: for long
// K from the forward, which kept them (k_gated_slopes reads them), else by computing them again with
// the gradients as the products' epilogue.  It then takes dx from K = [dg | du] and both
// weight gradients from M = [dg | du].
//
// Most cases run on square tiles of 256 or 128 (gated_wide.hip), projections of up to 64 rows on gated_skinny.hip's
// kernel, the backward of up to 15 columns on gated_narrow.hip's; here is what serves the others:
//
// k_tile: 64 x 64 tiles of any shape, stride and alignment, with 16x16 matrix instructions: fp32
// ones for fp32 (exact fp32 products), bf16/fp16 ones with fp32 sums.  A weight gradient's sum
// over rows is split over workgroups where there are few tiles; the parts are joined in order.
#include "gated.h"
#include "gated_narrow.h"
#include "gated_skinny.h"
#include "gated_wide.h"

namespace gsr {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// One matrix operand: element (i, k) at p[i * outer + k * inner], one of the strides 1.
template <typename T>
struct Operand {
  const T* p;
  int64_t stride;
};

template <typename T>
struct TileK {
  static constexpr int V = 16 / sizeof(T);    // elements of a 16-byte load
  static constexpr int BK = 4 * V;            // K of a step: 32 in 16 bits, 16 in fp32
  static constexpr int LD = BK + V;           // a row in shared memory, padded by 16 bytes
};

// One lane's piece of an operand's tile in flight (16 bytes of the type M that is multiplied, loaded as
// T), and where it goes in shared memory.  KC: K is the contiguous index.
template <typename M, typename T, bool KC>
__device__ __forceinline__ void tile_fetch(Operand<T> a, int64_t i0, int64_t rows, int64_t k0, int64_t k1,
                                           float (&v)[TileK<M>::V]) {
  constexpr int V = TileK<M>::V;
  const int t = threadIdx.x;
  if constexpr (KC) {
    const int64_t i = i0 + t / 4, k = k0 + (t % 4) * V;
    load_upto(a.p + i * a.stride + k, i < rows ? k1 - k : 0, v);
  } else {
    const int64_t k = k0 + t / (64 / V), i = i0 + (t % (64 / V)) * V;
    load_upto(a.p + k * a.stride + i, k < k1 ? rows - i : 0, v);
  }
}

template <typename T, bool KC>
__device__ __forceinline__ void tile_keep(T* lds, const float (&v)[TileK<T>::V]) {
  constexpr int V = TileK<T>::V, LD = TileK<T>::LD;
  const int t = threadIdx.x;
  if constexpr (KC) {
    store_vec(lds + (t / 4) * LD + (t % 4) * V, v);
  } else {
    const int k = t / (64 / V), i = (t % (64 / V)) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) lds[(i + j) * LD + k] = from_f<T>(v[j]);
  }
}

// c += a b over one step of K: a, b the 16 rows' 16 bytes of this lane (row lane % 16, K
// group lane / 16; the order of K is the same in both, so the sum does not care).
template <typename T>
__device__ __forceinline__ v4f tile_mma(const T* a, const T* b, v4f c);
template <>
__device__ __forceinline__ v4f tile_mma<bf16>(const bf16* a, const bf16* b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const v8bf*)a, *(const v8bf*)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ v4f tile_mma<f16>(const f16* a, const f16* b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const v8h*)a, *(const v8h*)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ v4f tile_mma<float>(const float* a, const float* b, v4f c) {
  const v4f x = *(const v4f*)a, y = *(const v4f*)b;
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s], y[s], c, 0, 0, 0);
  return c;
}

// acc[NB][nb][mb]: this wave's 32 x 32 of the tile (wave w: rows 32 (w % 2), columns 32 (w / 2)); a
// lane holds row m = 16 mb + lane % 16 and columns n = 16 nb + 4 (lane / 16) + 0..3.
// B(k): the operands for K step k0 (the gradient product changes matrices midway).
// TA, TB: the operands' types, MT: the type they are multiplied in.
template <typename MT, typename TA, typename TB, int NB, bool AKC, bool BKC, typename FB>
__device__ __forceinline__ void tile_product(Operand<TA> a, int64_t m0, int64_t M, FB b_at, int64_t n0, int64_t N,
                                             int64_t k0, int64_t k1, v4f (&acc)[NB][2][2]) {
  constexpr int V = TileK<MT>::V, BK = TileK<MT>::BK, LD = TileK<MT>::LD;
  __shared__ __attribute__((aligned(16))) MT as[64 * LD];
  __shared__ __attribute__((aligned(16))) MT bs[NB][64 * LD];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int at = (lane % 16) * LD + (lane / 16) * V, wm = wave % 2 * 32, wn = wave / 2 * 32;
#pragma unroll
  for (int q = 0; q < NB; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[q][i / 2][i % 2] = v4f{0.f, 0.f, 0.f, 0.f};
  float av[V], bv[NB][V];
  const auto fetch = [&](int64_t k) {
    tile_fetch<MT, TA, AKC>(a, m0, M, k, k1, av);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const auto o = b_at(q, k);
      tile_fetch<MT, TB, BKC>(o.op, n0, N, o.k, o.kend, bv[q]);
    }
  };
  if (k0 < k1) fetch(k0);
  for (int64_t k = k0; k < k1; k += BK) {
    __syncthreads();
    tile_keep<MT, AKC>(as, av);
#pragma unroll
    for (int q = 0; q < NB; ++q) tile_keep<MT, BKC>(bs[q], bv[q]);
    __syncthreads();
    if (k + BK < k1) fetch(k + BK);   // in flight over the products
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
          acc[q][nb][mb] = tile_mma<MT>(bs[q] + (wn + nb * 16) * LD + at, as + (wm + mb * 16) * LD + at, acc[q][nb][mb]);
  }
}

template <typename T>
struct OperandAt {
  Operand<T> op;
  int64_t k, kend;   // where the step's K lies in op, and its end there
};

// Forward (dgu NULL) or the gradients of the projections (h NULL): dgu [rows][2 gated_pad(hidden)],
// parts [row blocks][2][hidden] the column sums of each block of 64 rows (NULL: not wanted).
template <typename T, typename G>
__global__ __launch_bounds__(256) void k_tile_gated(const T* x, int64_t x_stride, const T* wg, const T* wu, const T* bg,
                                                    const T* bu, int act, GatedShape s, T* h, const T* dh,
                                                    int64_t dh_stride, G* dgu, float* parts) {
  const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
  v4f acc[2][2][2];
  tile_product<T, T, T, 2, true, true>(
      Operand<T>{x, x_stride}, m0, s.rows,
      [&](int q, int64_t k) { return OperandAt<T>{Operand<T>{q ? wu : wg, s.dim}, k, s.dim}; }, n0, s.hidden, 0, s.dim, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t pad = gated_pad(s.hidden);
  __shared__ float sums[2][2][64];   // [row half][dg, du][column]
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int64_t n = n0 + wave / 2 * 32 + nb * 16 + lane / 16 * 4, left = s.hidden - n;
    float gb[4], ub[4], sg[4] = {}, su[4] = {};
    load_upto(bg + n, bg ? left : 0, gb);
    load_upto(bu + n, bu ? left : 0, ub);
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const int64_t m = m0 + wave % 2 * 32 + mb * 16 + lane % 16;
      float g[4], u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[i] = acc[0][nb][mb][i] + gb[i];
        u[i] = acc[1][nb][mb][i] + ub[i];
      }
      float a[4], slope[4];
      activate<T>(act, g, a, slope);
      if (!dgu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = a[i] * u[i];
        if (m < s.rows) store_upto(h + m * s.hidden + n, left, g);
      } else if (m < s.rows) {
        float d[4];
        load_upto(dh + m * dh_stride + n, left, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i] = i < left ? d[i] * u[i] * slope[i] : 0.f;   // (the padding holds zeros)
          u[i] = i < left ? d[i] * a[i] : 0.f;
          sg[i] += g[i];
          su[i] += u[i];
        }
        store_vec(dgu + m * 2 * pad + n, g);   // n + 4 <= pad: the tiles cover the padding exactly
        store_vec(dgu + m * 2 * pad + pad + n, u);
      }
    }
    if (parts) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          sg[i] += __shfl_xor(sg[i], d);
          su[i] += __shfl_xor(su[i], d);
        }
        if (lane % 16 == 0) {
          const int c = wave / 2 * 32 + nb * 16 + lane / 16 * 4 + i;
          sums[wave % 2][0][c] = sg[i];
          sums[wave % 2][1][c] = su[i];
        }
      }
    }
  }
  if (parts) {
    __syncthreads();
    const int c = threadIdx.x % 64, which = threadIdx.x / 64;
    if (which < 2 && n0 + c < s.hidden)
      parts[((int64_t)blockIdx.x * 2 + which) * s.hidden + n0 + c] = sums[0][which][c] + sums[1][which][c];
  }
}

// dx = [dg | du] [Wg; Wu] over the columns of share blockIdx.z.  One share: into dx; more: fp32 parts
// [share][rows][dim].
template <typename T, typename G>
__global__ __launch_bounds__(256) void k_tile_dx(const G* dgu, const T* wg, const T* wu, GatedShape s, int64_t share, T* dx,
                                                 float* parts) {
  const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64, pad = gated_pad(s.hidden);
  const int64_t k0 = blockIdx.z * share, k1 = k0 + share < 2 * pad ? k0 + share : 2 * pad;
  v4f acc[1][2][2];
  tile_product<G, G, T, 1, true, false>(
      Operand<G>{dgu, 2 * pad}, m0, s.rows,
      [&](int, int64_t k) {
        return k < pad ? OperandAt<T>{Operand<T>{wg, s.dim}, k, s.hidden} : OperandAt<T>{Operand<T>{wu, s.dim}, k - pad, s.hidden};
      },
      n0, s.dim, k0, k1, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const int64_t m = m0 + wave % 2 * 32 + mb * 16 + lane % 16, n = n0 + wave / 2 * 32 + nb * 16 + lane / 16 * 4;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[0][nb][mb][i];
      if (m >= s.rows) continue;
      if (parts) {
        store_upto(parts + (blockIdx.z * s.rows + m) * s.dim + n, s.dim - n, v);
      } else {
        store_upto(dx + m * s.dim + n, s.dim - n, v);
      }
    }
}

// [dWg; dWu] = [dg | du]^T x over the rows of share blockIdx.z.  One share: into dwg, dwu; more:
// fp32 parts [share][2][hidden][dim].
template <typename T, typename G>
__global__ __launch_bounds__(256) void k_tile_dw(const G* dgu, const T* x, int64_t x_stride, GatedShape s, int64_t share,
                                                 T* dwg, T* dwu, float* parts) {
  const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64, pad = gated_pad(s.hidden);
  const int64_t k0 = blockIdx.z * share, k1 = k0 + share < s.rows ? k0 + share : s.rows;
  v4f acc[1][2][2];
  tile_product<G, G, T, 1, false, false>(
      Operand<G>{dgu, 2 * pad}, m0, 2 * pad,
      [&](int, int64_t k) { return OperandAt<T>{Operand<T>{x, x_stride}, k, k1}; }, n0, s.dim, k0, k1, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const int64_t c = m0 + wave % 2 * 32 + mb * 16 + lane % 16, n = n0 + wave / 2 * 32 + nb * 16 + lane / 16 * 4;
      const int which = c >= pad;
      const int64_t m = c - which * pad;
      if (m >= s.hidden) continue;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[0][nb][mb][i];
      if (parts) {
        store_upto(parts + ((blockIdx.z * 2 + which) * s.hidden + m) * s.dim + n, s.dim - n, v);
      } else if (T* to = which ? dwu : dwg) {
        store_upto(to + m * s.dim + n, s.dim - n, v);
      }
    }
}

// [a | b], a the first `split` of n values, = the sum over `count` rows of parts [count][n]: GROUPS
// lanes a value, each a fixed share of the rows with loads in flight, then the lanes in order.
template <typename T, int GROUPS>
__global__ __launch_bounds__(GROUPS == 1 ? 256 : GROUPS * 64) void k_gated_join(const float* parts, int64_t count, int64_t n,
                                                                                int64_t split, T* a, T* b) {
  constexpr int COLS = GROUPS == 1 ? 256 : 64;
  __shared__ float sum[GROUPS][GROUPS == 1 ? 1 : 65];
  const int lane = threadIdx.x % COLS, grp = threadIdx.x / COLS;
  const int64_t c = (int64_t)blockIdx.x * COLS + lane;
  float s = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int64_t r = grp; r < count; r += GROUPS) s += parts[r * n + c];
  }
  if constexpr (GROUPS > 1) {
    sum[grp][lane] = s;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) s += sum[k][lane];
  }
  if (c < split) {
    if (a) a[c] = from_f<T>(s);
  } else if (c < n && b) {
    b[c - split] = from_f<T>(s);
  }
}

template <typename T>
static void gated_join(const float* parts, int64_t count, int64_t n, int64_t split, void* a, void* b, hipStream_t st) {
  if (count < 16) {
    k_gated_join<T, 1><<<(unsigned)ceil_div64(n, 256), 256, 0, st>>>(parts, count, n, split, (T*)a, (T*)b);
  } else {
    k_gated_join<T, 16><<<(unsigned)ceil_div64(n, 64), 1024, 0, st>>>(parts, count, n, split, (T*)a, (T*)b);
  }
}

// The gradients of the projections from what the forward kept: dgu, and parts [blocks of `each` rows][2]
// [hidden] of the column sums (NULL: not wanted).  Bound by memory: 12 bytes an element in 16 bits, 20 in
// fp32 (8 columns a lane, 256 a workgroup; 16384 x 5632 bf16 228 us, 4.9 TB/s).
template <typename T, typename G>
__global__ __launch_bounds__(256) void k_gated_slopes(const void* saved, const T* dh, int64_t dh_stride, int act, GatedShape s,
                                                      int each, G* dgu, float* parts) {
  const int64_t pad = gated_pad(s.hidden);
  const uint32_t across = (uint32_t)((pad + 255) / 256), block = blockIdx.x / across;   // (rows may be more than a grid's second side)
  const int64_t n0 = (int64_t)(blockIdx.x % across) * 256, n = n0 + threadIdx.x % 32 * 8, left = s.hidden - n;
  const Kept<T> kept((void*)saved, s.rows, s.hidden);
  const int64_t m0 = (int64_t)block * each + threadIdx.x / 32;
  float sg[8] = {}, su[8] = {};
  if (n < pad) {
#pragma unroll 2
    for (int r = 0; r < each; r += 8) {
      const int64_t m = m0 + r;
      if (m >= s.rows) break;
      float g[8], u[8], d[8];
      kept.load(m * pad + n, g, u);
      load_upto(dh + m * dh_stride + n, left, d);
      float a[8], slope[8];
      activate<T>(act, g, a, slope);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[i] = i < left ? d[i] * u[i] * slope[i] : 0.f;   // (the padding holds zeros)
        u[i] = i < left ? d[i] * a[i] : 0.f;
        sg[i] += g[i];
        su[i] += u[i];
      }
      store_vec(dgu + m * 2 * pad + n, g);
      store_vec(dgu + m * 2 * pad + pad + n, u);
    }
  }
  if (!parts) return;
  __shared__ float sum[8][2][256 + 8];
  const int c = threadIdx.x % 32 * 8, rl = threadIdx.x / 32;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum[rl][0][c + i] = sg[i];
    sum[rl][1][c + i] = su[i];
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int64_t col = n0 + threadIdx.x;
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) v += sum[r][which][threadIdx.x];
    if (col < s.hidden) parts[((int64_t)block * 2 + which) * s.hidden + col] = v;
  }
}

// Rows of its workgroups: 64, fewer where that makes less than two workgroups a CU (777 x 1363 bf16 4.9 us
// against 9.1).
static int gated_slopes_rows(GatedShape s) {
  int each = 64;
  while (each > 8 && ceil_div64(gated_pad(s.hidden), 256) * ceil_div64(s.rows, each) < 512) each /= 2;
  return each;
}

// Shares of K in a product of `tiles` 64 x 64 tiles: enough workgroups for two a CU, each share at
// least 128 of K, the fp32 parts of `values` results at most 64 MB.
static int64_t gated_shares(int64_t tiles, int64_t k, int64_t values) {
  int64_t n = 512 / tiles;
  n = n < k / 128 ? n : k / 128;
  const int64_t most = (64 << 20) / 4 / values;
  n = n < most ? n : most;
  return n < 1 ? 1 : n;
}

// Padded copies of up to three matrices: to [rows][kdim] = p [rows][dim] (row stride `stride`) and
// zeros, rows that start at 16 bytes and are whole 16-byte pieces.
template <typename T>
struct GatedPads {
  const T* p[3];
  T* to[3];
  int64_t rows[3], stride[3];   // rows 0: none
  int64_t dim, kdim;
};

template <typename T>
__global__ __launch_bounds__(256) void k_gated_pad(GatedPads<T> a) {
  constexpr int V = 16 / sizeof(T);
  const int64_t per = a.kdim / V;
  int64_t first = 0;
#pragma unroll
  for (int q = 0; q < 3; ++q) {   // one run of pieces through all three
    const int64_t n = a.rows[q] * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < first + n; i += (int64_t)gridDim.x * 256) {
      if (i < first) continue;
      const int64_t r = (i - first) / per, c = (i - first) % per * V;
      float v[V];
      load_upto(a.p[q] + r * a.stride[q] + c, a.dim - c, v);
      store_vec(a.to[q] + r * a.kdim + c, v);
    }
    first += n;
  }
}

// Tile side of a product of rows x cols outputs over k.  256 (16 bits) where every CU gets at least 96
// steps of K: 16384 x 2048 -> 5632, at 352 a CU, forward 660 us against 726 with 128, dW 593
// against 877; at 88 the two are within 5 %; at 31 (16000 x 512 -> 2048) 111 us against 101.
// 64 (any alignment, no padded copies) for dims whose K is hardly a step, and dx and dW of 64 columns,
// half a tile; and where 128 has fewer than two steps a CU, its tiles cut along K as well, in fp32 or
// with few rows.  Forward and backward, 128 against 64: fp32 500 x 1000 -> 1000 100 us against 190, 256
// x 1024 -> 2816 128 against 197, 16000 x 128 -> 256 105 against 126; 200 x 100 -> 1000 59 against 43,
// 2000 x 128 -> 128 52 against 48; dx of 16 x 2048 -> 4096 bf16 19 us against 25, of 40 x 1024 ->
// 2816 14.5 against 14.0.
static bool gated_pads_few(int type, GatedShape s);
static int gated_side(int type, int64_t rows, int64_t cols, int64_t k, GatedShape s) {
  const bool few = s.rows <= kSkinnyRows;
  if (s.dim < 64 || (few && s.dim % 8 && !gated_pads_few(type, s))) return 64;
  const int64_t steps = gated_wide_steps(type, k);
  if (type == GSR_F32 && cols <= 64) return 64;
  if (type == GSR_F32 || few) return ceil_div64(rows, 128) * ceil_div64(cols, 128) * steps >= 512 ? 128 : 64;
  return ceil_div64(rows, 256) * ceil_div64(cols, 256) * steps >= 256 * 96 ? 256 : 128;
}

// What a wide case's operands need: rows of whole 16-byte pieces at 16-byte addresses, 256 of them
// within 31 bits.
template <typename T>
static bool gated_aligned(const T* p, int64_t dim, int64_t stride) {
  constexpr int V = 16 / sizeof(T);
  return (uintptr_t)p % 16 == 0 && dim % V == 0 && stride % V == 0 && stride <= 1 << 20;
}

// The least dim whose forward keeps its projections for the backward (on tiles of 128 and 256): what that
// moves, 12 bytes an element (16 in fp32), does not grow with dim, what it saves does.  Forward and
// gradients of the projections, kept against computed again: 16384 x 2048 -> 5632 bf16 915 us against
// 1487, 4096 x 256 -> 2816 55 against 62, x 128 50 against 54 and not worth its memory; fp32 4096 x
// 128 -> 2816 111 against 146.
static bool gated_keeps(int type, int64_t dim) { return dim >= (type == GSR_F32 ? 128 : 256); }

// Whether few rows' operands are copied to whole 16-byte pieces: 16-bit weights of odd rows, which the kernel for few
// rows would read at 0.8 TB/s, large enough for the copy's launch to pay (60 x 2699 -> 5750 bf16,
// forward and backward: 98 us against 266).
static bool gated_pads_few(int type, GatedShape s) {
  return s.rows <= kSkinnyRows && type != GSR_F32 && s.dim % 8 && s.hidden * s.dim >= 1 << 21;
}

// Whether a 16-bit block's backward keeps the projections' gradients in fp32 and multiplies them so: where
// products are short (in 64 x 64 tiles 2^24 products, a few us at the fp32 rate) or dx has few
// values.  There one more rounding to 16 bits need not average out: the root mean square error of
// a gradient grows by up to 2.1, that of larger ones by 1.4.  (65 x 256 -> 512 bf16: 30 us against 25;
// 4096 x 256 -> 256, left in 16 bits, would take 66 against 33.)
static bool gated_exact(int type, GatedShape s) {
  if (type == GSR_F32) return false;
  const int64_t r = s.rows < 64 ? 64 : s.rows, d = s.dim < 64 ? 64 : s.dim;
  return r * d <= (1 << 24) / s.hidden || s.rows * s.dim <= 2048;
}

// How a pass is laid out: each product's tile side, the 64 x 64 tiles' shares of K, and its workspace (byte
// offsets).  There is room for padded copies wherever a wide product may need them: an odd dim, rows
// or addresses that are not multiples of 16 bytes.
struct GatedPlan {
  int fwd, dx, dw;               // tile sides
  bool beside;                   // dx and dW run side by side
  bool keep;                     // the forward keeps its projections
  bool keep_pads;                // and the padded copies of x and the weights, where dim is the reason for them
  int64_t kept_pads, kept;       // their place behind the projections; bytes in all
  bool exact;                    // the backward's products take the projections' gradients in fp32
  int64_t n_dx, n_dw;            // shares
  WideRounds r_fwd, r_dx, r_dw;  // and those of the wide products
  int64_t kdim;                  // dim in whole 16-byte pieces
  int64_t x, wg, wu, cuts, dgu, bias, bias_rows, dx_parts, dw_parts, total;   // (cuts: the forward's)
};

// Whether the backward is one kernel (gated_narrow.hip).
static bool gated_is_narrow(GatedShape s) { return s.dim <= kNarrowDim; }

static GatedPlan gated_plan(GatedShape s, int type, bool backward) {
  GatedPlan w{};
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (backward && gated_is_narrow(s)) {
    const NarrowPlan n = gated_narrow_plan(s);
    w.dw_parts = take(n.dw_floats(s) * 4);
    w.dx_parts = take(n.dx_floats(s) * 4);
    w.total = at;
    return w;
  }
  const int64_t pad = gated_pad(s.hidden);
  w.fwd = gated_side(type, s.rows, 2 * pad, s.dim, s);
  // (fp32's forward: from eight steps on, which shares of two cut well; 325 x 592 -> 398 19 us against 37 in 64 x 64
  // tiles, and its backward 34 against 68, from kept projections)
  if (type == GSR_F32 && s.rows > kSkinnyRows && gated_wide_steps(type, s.dim) >= 8) w.fwd = 128;
  w.exact = gated_exact(type, s);
  w.dx = w.exact ? 64 : gated_side(type, s.rows, s.dim, 2 * pad, s);
  w.dw = w.exact ? 64 : gated_side(type, 2 * pad, s.dim, s.rows, s);
  const int64_t es = (int64_t)type_size(type), piece = 16 / es;
  w.kdim = (s.dim + piece - 1) / piece * piece;
  const int64_t rb = ceil_div64(s.rows, 64), hb = 2 * pad / 64, db = ceil_div64(s.dim, 64);
  w.n_dx = w.dx > 64 ? 1 : gated_shares(rb * db, 2 * pad, s.rows * s.dim);
  w.n_dw = w.dw > 64 ? 1 : gated_shares(hb * db, s.rows, 2 * s.hidden * s.dim);
  const auto tiles = [](int side, int64_t r, int64_t c) { return ceil_div64(r, side) * ceil_div64(c, side); };
  const int64_t x_steps = gated_wide_steps(type, 2 * pad), w_steps = gated_wide_steps(type, s.rows);
  WideRounds r[2];
  w.beside = w.dx == 128 && w.dw == 128 &&
             gated_wide_back_rounds(type, {tiles(128, s.rows, s.dim), tiles(128, 2 * pad, s.dim)}, {x_steps, w_steps}, r);
  if (w.beside) {
    w.r_dx = r[0], w.r_dw = r[1];
  } else {
    if (w.dx > 64) w.r_dx = gated_wide_rounds(type, w.dx, ceil_div64(s.rows, w.dx), ceil_div64(s.dim, w.dx), x_steps);
    if (w.dw > 64) w.r_dw = gated_wide_rounds(type, w.dw, ceil_div64(2 * pad, w.dw), ceil_div64(s.dim, w.dw), w_steps);
  }
  if (s.rows <= kSkinnyRows) w.fwd = 64;   // (the kernel for few rows)
  const bool pads = w.fwd > 64 || gated_pads_few(type, s);
  const bool xw = pads || (backward && w.dw > 64), ww = pads || (backward && w.dx > 64);
  w.x = take(xw ? s.rows * w.kdim * es : 0);
  w.wg = take(ww ? s.hidden * w.kdim * es : 0);
  w.wu = take(ww ? s.hidden * w.kdim * es : 0);
  if (w.fwd > 64)
    w.r_fwd = gated_wide_rounds(type, w.fwd, ceil_div64(s.rows, w.fwd), ceil_div64(pad, w.fwd / 2), gated_wide_steps(type, s.dim));
  w.cuts = take(w.fwd > 64 && !backward ? w.r_fwd.bytes(w.fwd) : 0);
  w.keep = (w.fwd > 64 || s.rows <= kSkinnyRows) && gated_keeps(type, s.dim);
  w.keep_pads = pads && w.kdim != s.dim && (w.dx > 64 || w.dw > 64 || (w.fwd > 64 && !w.keep));   // (what reads them)
  w.kept_pads = !w.keep ? 0 : type == GSR_F32 ? Kept<float>::bytes(s.rows, s.hidden) : Kept<bf16>::bytes(s.rows, s.hidden);
  w.kept = w.kept_pads + (w.keep_pads ? (s.rows + 2 * s.hidden) * w.kdim * es : 0);
  w.bias_rows = s.rows <= kSkinnyRows ? 1 : w.fwd > 64 ? ceil_div64(s.rows, w.fwd) * 2 : rb;
  w.dgu = take(backward ? s.rows * 2 * pad * (w.exact ? 4 : es) : 0);
  const int64_t kept_rows = w.keep ? ceil_div64(s.rows, gated_slopes_rows(s)) : 0;
  w.bias = take(backward ? (kept_rows > w.bias_rows ? kept_rows : w.bias_rows) * 2 * s.hidden * 4 : 0);
  w.dx_parts = take(!backward ? 0 : w.dx > 64 ? w.r_dx.bytes(w.dx) : w.n_dx > 1 ? w.n_dx * s.rows * s.dim * 4 : 0);
  w.dw_parts = take(!backward  ? 0
                    : w.dw > 64 ? w.r_dw.bytes(w.dw)
                    : w.n_dw > 1 ? w.n_dw * 2 * s.hidden * s.dim * 4
                                 : 0);
  w.total = at;
  return w;
}

// The wide products' operands, copied into whole 16-byte pieces where they are not: for the backward too
// (`pads`, NULL: not wanted) or in the workspace.  `made`: pads holds the copies already.
template <typename T>
static GatedWide gated_wide_args(const T* x, int64_t x_stride, const T* wg, const T* wu, const void* bg, const void* bu, int act,
                                 GatedShape s, const GatedPlan& w, bool use_x, bool use_w, char* ws, T* pads, bool made,
                                 hipStream_t st) {
  GatedWide a{};
  a.s = s;
  a.kdim = w.kdim, a.x_stride = x_stride, a.w_stride = s.dim;
  a.x = x, a.wg = wg, a.wu = wu, a.bg = bg, a.bu = bu, a.act = act;
  GatedPads<T> p{};
  p.dim = s.dim, p.kdim = w.kdim;
  if (use_x && !gated_aligned(x, s.dim, x_stride)) {
    p.p[0] = x, p.to[0] = pads ? pads : (T*)(ws + w.x), p.rows[0] = s.rows, p.stride[0] = x_stride;
    a.x = p.to[0], a.x_stride = w.kdim;
  }
  if (use_w && !(gated_aligned(wg, s.dim, s.dim) && gated_aligned(wu, s.dim, s.dim))) {
    T* const to = pads ? pads + s.rows * w.kdim : nullptr;
    p.p[1] = wg, p.to[1] = to ? to : (T*)(ws + w.wg), p.rows[1] = s.hidden, p.stride[1] = s.dim;
    p.p[2] = wu, p.to[2] = to ? to + s.hidden * w.kdim : (T*)(ws + w.wu), p.rows[2] = s.hidden, p.stride[2] = s.dim;
    a.wg = p.to[1], a.wu = p.to[2], a.w_stride = w.kdim;
  }
  if (made) return a;
  const int64_t pieces = (p.rows[0] + p.rows[1] + p.rows[2]) * (w.kdim / (16 / (int64_t)sizeof(T))), blocks = ceil_div64(pieces, 256);
  if (pieces) k_gated_pad<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, st>>>(p);
  return a;
}

template <typename T>
static constexpr int type_of() {
  return __is_same(T, float) ? GSR_F32 : __is_same(T, bf16) ? GSR_BF16 : GSR_F16;
}

template <typename T>
static void gated_fwd(const T* x, int64_t x_stride, const T* wg, const T* wu, const T* bg, const T* bu, int act, GatedShape s,
                      T* h, void* kept, char* ws, hipStream_t st) {
  const int type = type_of<T>();
  const GatedPlan w = gated_plan(s, type, false);
  T* const pads = kept && w.keep_pads ? (T*)((char*)kept + w.kept_pads) : nullptr;
  if (s.rows <= kSkinnyRows) {
    GatedSkinny f{s, x, wg, wu, bg, bu, nullptr, x_stride, 0, h, nullptr, nullptr, act, false, w.keep ? kept : nullptr};
    // (up to 16 rows the copy pays with a backward to follow: 1 x 4095 -> 11264 bf16 forward alone 77 us without it, 122
    // with; with the backward 495 and 238)
    if (gated_pads_few(type, s) && (pads || s.rows > 16)) {
      const GatedWide a = gated_wide_args<T>(x, x_stride, wg, wu, bg, bu, act, s, w, true, true, ws, pads, false, st);
      f.s.dim = w.kdim, f.x = a.x, f.x_stride = a.x_stride, f.wg = a.wg, f.wu = a.wu;
    }
    gated_skinny(type, f, st);
    return;
  }
  if (w.fwd > 64) {
    GatedWide a = gated_wide_args<T>(x, x_stride, wg, wu, bg, bu, act, s, w, true, true, ws, pads, false, st);
    a.h = h, a.kept = w.keep ? kept : nullptr, a.cuts = (float*)(ws + w.cuts);
    gated_wide(type, kWideFwd, w.fwd, a, w.r_fwd, st);
    return;
  }
  const dim3 grid((unsigned)ceil_div64(s.rows, 64), (unsigned)ceil_div64(s.hidden, 64));
  k_tile_gated<T, T><<<grid, 256, 0, st>>>(x, x_stride, wg, wu, bg, bu, act, s, h, nullptr, 0, nullptr, nullptr);
}

// G: the type that the projections' gradients are kept and multiplied in.
template <typename T, typename G>
static void gated_bwd_as(const T* x, int64_t x_stride, const T* wg, const T* wu, const T* bg, const T* bu, int act, GatedShape s,
                      const T* dh, int64_t dh_stride, const void* kept, T* dx, T* dwg, T* dwu, T* dbg, T* dbu, char* ws,
                      hipStream_t st) {
  const int type = type_of<T>();
  GatedPlan w = gated_plan(s, type, true);
  const int64_t rb = ceil_div64(s.rows, 64), db = ceil_div64(s.dim, 64), pad = gated_pad(s.hidden);
  const bool weights = dwg || dwu, few = s.rows <= kSkinnyRows, keep = w.keep && kept;
  const int each = gated_slopes_rows(s);
  if (keep) w.bias_rows = ceil_div64(s.rows, each);
  G* dgu = (G*)(ws + w.dgu);
  float* bias = dbg || dbu ? (float*)(ws + w.bias) : nullptr;
  GatedWide a{};
  if (w.fwd > 64 || w.dx > 64 || w.dw > 64) {
    const bool again = w.fwd > 64 && !keep;   // both projections are computed again
    T* const pads = kept && w.keep_pads ? (T*)((char*)kept + w.kept_pads) : nullptr;
    a = gated_wide_args<T>(x, x_stride, wg, wu, bg, bu, act, s, w, again || (weights && w.dw > 64), again || (dx && w.dx > 64), ws,
                           pads, pads != nullptr, st);
    a.dh = dh, a.dh_stride = dh_stride, a.dgu = dgu, a.dgu32 = w.exact, a.dx = dx, a.dwg = dwg, a.dwu = dwu;
  }
  if (keep) {
    k_gated_slopes<T, G><<<(unsigned)(ceil_div64(pad, 256) * w.bias_rows), 256, 0, st>>>(kept, dh, dh_stride, act, s, each, dgu, bias);
  } else if (few) {
    gated_skinny(type, GatedSkinny{s, x, wg, wu, bg, bu, dh, x_stride, dh_stride, nullptr, dgu, bias, act, w.exact}, st);
  } else if (w.fwd > 64) {
    a.parts = bias;
    gated_wide(type, kWideGrad, w.fwd, a, w.r_fwd, st);
  } else {
    k_tile_gated<T, G><<<dim3((unsigned)rb, (unsigned)(pad / 64)), 256, 0, st>>>(x, x_stride, wg, wu, bg, bu, act, s, nullptr, dh,
                                                                            dh_stride, dgu, bias);
  }
  if (bias) gated_join<T>(bias, w.bias_rows, 2 * s.hidden, s.hidden, dbg, dbu, st);
  if (dx && weights && w.beside) {
    gated_wide_back(type, a, w.r_dx, (float*)(ws + w.dx_parts), w.r_dw, (float*)(ws + w.dw_parts), st);
    return;
  }
  if (dx) {
    const int64_t n = w.n_dx, share = ceil_div64(ceil_div64(2 * pad, n), 64) * 64;
    float* parts = n > 1 ? (float*)(ws + w.dx_parts) : nullptr;
    if (w.dx > 64) {
      a.cuts = (float*)(ws + w.dx_parts);
      gated_wide(type, kWideDx, w.dx, a, w.r_dx, st);
    } else {
      k_tile_dx<T, G><<<dim3((unsigned)rb, (unsigned)db, (unsigned)n), 256, 0, st>>>(dgu, wg, wu, s, share, dx, parts);
    }
    if (parts) gated_join<T>(parts, n, s.rows * s.dim, s.rows * s.dim, dx, nullptr, st);
  }
  if (weights) {
    const int64_t n = w.n_dw, share = ceil_div64(ceil_div64(s.rows, n), 64) * 64;
    float* parts = n > 1 ? (float*)(ws + w.dw_parts) : nullptr;
    if (w.dw > 64) {
      a.cuts = (float*)(ws + w.dw_parts);
      gated_wide(type, kWideDw, w.dw, a, w.r_dw, st);
    } else {
      k_tile_dw<T, G><<<dim3((unsigned)(2 * pad / 64), (unsigned)db, (unsigned)n), 256, 0, st>>>(dgu, x, x_stride, s, share, dwg,
                                                                                              dwu, parts);
    }
    if (parts) gated_join<T>(parts, n, 2 * s.hidden * s.dim, s.hidden * s.dim, dwg, dwu, st);
  }
}

template <typename T>
static void gated_bwd(const T* x, int64_t x_stride, const T* wg, const T* wu, const T* bg, const T* bu, int act, GatedShape s,
                      const T* dh, int64_t dh_stride, const void* kept, T* dx, T* dwg, T* dwu, T* dbg, T* dbu, char* ws,
                      hipStream_t st) {
  if (gated_is_narrow(s)) {
    const GatedPlan w = gated_plan(s, type_of<T>(), true);
    GatedNarrow a{s, x, wg, wu, bg, bu, dh, x_stride, dh_stride, act, dx, dwg, dwu, dbg, dbu};
    a.dw_parts = (float*)(ws + w.dw_parts), a.dx_parts = (float*)(ws + w.dx_parts);
    gated_narrow(type_of<T>(), a, st);
  } else if (gated_exact(type_of<T>(), s)) {
    gated_bwd_as<T, float>(x, x_stride, wg, wu, bg, bu, act, s, dh, dh_stride, kept, dx, dwg, dwu, dbg, dbu, ws, st);
  } else {
    gated_bwd_as<T, T>(x, x_stride, wg, wu, bg, bu, act, s, dh, dh_stride, kept, dx, dwg, dwu, dbg, dbu, ws, st);
  }
}

static int gated_check(const char* who, GatedShape s, int64_t x_stride, int type, int act) {
  GSR_REQUIRE(s.rows >= 0 && s.rows <= (int64_t)1 << 26, "%s: bad rows %lld", who, (long long)s.rows);
  GSR_REQUIRE(s.dim >= 1 && s.dim <= 1 << 20 && s.hidden >= 1 && s.hidden <= 1 << 20, "%s: bad dim %lld or hidden %lld", who,
              (long long)s.dim, (long long)s.hidden);
  GSR_REQUIRE(s.rows <= 1 || x_stride >= s.dim, "%s: row stride %lld below dim %lld", who, (long long)x_stride,
              (long long)s.dim);
  GSR_REQUIRE(known_type(type), "%s: bad type %d", who, type);
  GSR_REQUIRE(act >= GSR_ACT_SILU && act <= GSR_ACT_SIGMOID, "%s: bad activation %d", who, act);
  return 0;
}

}  // namespace gsr

using namespace gsr;

extern "C" size_t gsr_gated_workspace(int64_t rows, int64_t dim, int64_t hidden, int32_t type, int32_t backward) {
  const GatedShape s{rows, dim, hidden};
  if (gated_check("gsr_gated_workspace", s, dim, type, GSR_ACT_SILU) || rows == 0) return 0;
  return (size_t)gated_plan(s, type, backward != 0).total;
}

extern "C" size_t gsr_gated_kept(int64_t rows, int64_t dim, int64_t hidden, int32_t type) {
  const GatedShape s{rows, dim, hidden};
  if (gated_check("gsr_gated_kept", s, dim, type, GSR_ACT_SILU) || rows == 0) return 0;
  return (size_t)gated_plan(s, type, false).kept;
}

extern "C" int gsr_gated_fwd(const void* x, int64_t rows, int64_t dim, int64_t x_stride, int32_t type, const void* wg,
                             const void* wu, int64_t hidden, const void* bg, const void* bu, int32_t act, void* h,
                             void* kept, void* workspace, size_t workspace_bytes, void* stream) {
  const GatedShape s{rows, dim, hidden};
  if (const int e = gated_check("gsr_gated_fwd", s, x_stride, type, act)) return e;
  if (rows == 0) return 0;
  GSR_REQUIRE(x && wg && wu && h, "gsr_gated_fwd: null pointer");
  GSR_REQUIRE(!bg == !bu, "gsr_gated_fwd: bg and bu go together");
  GSR_REQUIRE(workspace_bytes >= gsr_gated_workspace(rows, dim, hidden, type, 0) && (workspace || workspace_bytes == 0),
              "gsr_gated_fwd: workspace too small (%zu bytes)", workspace_bytes);
  GSR_REQUIRE(((uintptr_t)workspace | (uintptr_t)kept) % 256 == 0, "gsr_gated_fwd: workspace and kept must start at 256 bytes");
  char* ws = (char*)workspace;
  const auto st = (hipStream_t)stream;
  if (type == GSR_F32) {
    gated_fwd((const float*)x, x_stride, (const float*)wg, (const float*)wu, (const float*)bg, (const float*)bu, act, s, (float*)h, kept, ws, st);
  } else if (type == GSR_BF16) {
    gated_fwd((const bf16*)x, x_stride, (const bf16*)wg, (const bf16*)wu, (const bf16*)bg, (const bf16*)bu, act, s, (bf16*)h, kept, ws, st);
  } else {
    gated_fwd((const f16*)x, x_stride, (const f16*)wg, (const f16*)wu, (const f16*)bg, (const f16*)bu, act, s, (f16*)h, kept, ws, st);
  }
  GSR_LAUNCH_CHECK("gsr_gated_fwd");
  return 0;
}

extern "C" int gsr_gated_bwd(const void* x, int64_t rows, int64_t dim, int64_t x_stride, int32_t type, const void* wg,
                             const void* wu, int64_t hidden, const void* bg, const void* bu, int32_t act, const void* dh,
                             int64_t dh_stride, const void* kept, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const GatedShape s{rows, dim, hidden};
  if (const int e = gated_check("gsr_gated_bwd", s, x_stride, type, act)) return e;
  GSR_REQUIRE(rows <= 1 || dh_stride >= hidden, "gsr_gated_bwd: dh row stride %lld below hidden", (long long)dh_stride);
  GSR_REQUIRE(wg && wu && (rows == 0 || (x && dh)), "gsr_gated_bwd: null pointer");
  GSR_REQUIRE(!bg == !bu, "gsr_gated_bwd: bg and bu go together");
  GSR_REQUIRE(workspace_bytes >= gsr_gated_workspace(rows, dim, hidden, type, 1) && (workspace || workspace_bytes == 0),
              "gsr_gated_bwd: workspace too small (%zu bytes)", workspace_bytes);
  GSR_REQUIRE(((uintptr_t)workspace | (uintptr_t)kept) % 256 == 0, "gsr_gated_bwd: workspace and kept must start at 256 bytes");
  const auto st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (rows == 0) {   // sums over no rows
    const auto zero = [&](void* p, int64_t n) {
      const int64_t most = 1 << 30;   // (a launch holds less than 2^32 threads, one a value)
      for (int64_t at = 0; p && at < n; at += most)
        gated_join<bf16>(nullptr, 0, n - at < most ? n - at : most, most, (bf16*)p + at, nullptr, st);
    };
    const int64_t each = type == GSR_F32 ? 2 : 1;   // zeros of any type, 16 bits at a time
    zero(dwg, hidden * dim * each);
    zero(dwu, hidden * dim * each);
    zero(dbg, hidden * each);
    zero(dbu, hidden * each);
  } else if (type == GSR_F32) {
    gated_bwd((const float*)x, x_stride, (const float*)wg, (const float*)wu, (const float*)bg, (const float*)bu, act, s, (const float*)dh,
              dh_stride, kept, (float*)dx, (float*)dwg, (float*)dwu, (float*)dbg, (float*)dbu, ws, st);
  } else if (type == GSR_BF16) {
    gated_bwd((const bf16*)x, x_stride, (const bf16*)wg, (const bf16*)wu, (const bf16*)bg, (const bf16*)bu, act, s, (const bf16*)dh,
              dh_stride, kept, (bf16*)dx, (bf16*)dwg, (bf16*)dwu, (bf16*)dbg, (bf16*)dbu, ws, st);
  } else {
    gated_bwd((const f16*)x, x_stride, (const f16*)wg, (const f16*)wu, (const f16*)bg, (const f16*)bu, act, s, (const f16*)dh,
              dh_stride, kept, (f16*)dx, (f16*)dwg, (f16*)dwu, (f16*)dbg, (f16*)dbu, ws, st);
  }
  GSR_LAUNCH_CHECK("gsr_gated_bwd");
  return 0;
}
