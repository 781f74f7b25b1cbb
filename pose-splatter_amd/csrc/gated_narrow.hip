// The gated block's backward pass for narrow inputs (dim <= 15), in one kernel and a join: its products are
// short in one direction, so what passes through memory decides.
//
// dh is read once and the projections' gradients are not written: a wave holds 64 rows of x in
// registers, and goes through its columns of the projections 16 at a time.  For 16 rows of them
//   g, u = x W^T + b             4 columns of g and u a lane, for its row of x
//   dg, du                       in registers, from dh
//   dx += dg Wg + du Wu          dg and du are the instruction's operand as they are: K's order is
//                                free, and lane group q's four columns are K = q of four instructions
//   [dW db] += [dg du]^T [x 1]   sums over rows: dg and du turned through 16 x 16 of shared memory; the
//                                column of ones next to x's own sums the biases' gradients
// All in fp32, by 16x16x4 matrix instructions, whatever the type.  The waves of a workgroup share dx
// through shared memory; the rows' parts of dW (and dx's, of workgroups that share rows) go through
// memory and are joined in order.
//
// Against projections, dx and dW as products of their own (gated.hip), 16000 rows, fp32: 8 -> 128 18 us
// (38), 8 -> 12288 582 us (2515), 15 -> 2000 125 us (410); bf16 18 (31), 504 (1908), 115 (320); 65 x
// 3 -> 100 13 us (22), 1 x 8 -> 12288 15 us (18).  At 8 -> 12288 it waits for the activation's vector
// instructions (290 us of fp32), then for the weights' parts (217 us).  Two blocks of 16 columns do
// not fit the registers: 30 -> 512 would take 144 us against 102.
#include "gated_narrow.h"

namespace gsr {

typedef float nv4f __attribute__((ext_vector_type(4)));

constexpr int kNarrowWaves = 8, kNarrowRows = 64, kTurn = 20;   // kTurn: floats a row, so that both accesses spread over the banks

// Four neighbouring elements as they lie in memory, to be in flight while others are worked on.
template <typename T>
struct Four {
  uint32_t w[sizeof(T)];
  __device__ __forceinline__ void load(const T* p, int64_t n) {   // the first n, then zeros
    if (n >= 4) {
      const Pack<uint32_t, sizeof(T)> k = *reinterpret_cast<const Pack<uint32_t, sizeof(T)>*>(p);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) w[i] = k.v[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4) {
          w[i] = __builtin_bit_cast(uint32_t, p[i]);
        } else {
          w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i % 2));
        }
      }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      return to_f(__builtin_bit_cast(T, (uint16_t)(i % 2 ? w[i / 2] >> 16 : w[i / 2])));
    }
  }
};

__device__ __forceinline__ nv4f narrow_mma(float a, float b, nv4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// KS: steps of 4 of dim.
template <typename T, int KS>
__global__ __launch_bounds__(kNarrowWaves * 64) void k_narrow(GatedNarrow a) {
  constexpr int LD = 17, EACH = KS;   // floats a row of dx's sums; elements of 16 rows of W a lane
  constexpr int WAVE = 2 * 2 * 16 * kTurn, TURNS = kNarrowWaves * WAVE, SUMS = kNarrowWaves * kNarrowRows * LD;
  __shared__ __attribute__((aligned(16))) float lds[TURNS > SUMS ? TURNS : SUMS];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l = lane % 16, q = lane / 16;
  float* const turn = lds + wave * WAVE;            // the wave's own: a wave reads and writes shared memory in order
  float* const wrow = turn + 2 * 16 * kTurn;        // its 16 rows of both weights
  const GatedShape s = a.s;
  const int64_t c0 = blockIdx.y * a.cols, c1 = c0 + a.cols < s.hidden ? c0 + a.cols : s.hidden;
  const int blocks = (int)((c1 - c0 + 15) / 16), dim = (int)s.dim, width = (dim + 4) / 4 * 4;
  const bool weights = a.dwg || a.dwu || a.dbg || a.dbu;
  const auto x_at = [&](int64_t r, int d) {   // element d of row r of [x 1]
    return r >= s.rows || d > dim ? 0.f : d == dim ? 1.f : to_f(((const T*)a.x)[r * a.x_stride + d]);
  };
  int w_to[EACH];   // where the lane's elements of 16 rows of W go
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int e = lane + j * 64;
    w_to[j] = e < 16 * dim ? e / dim * kTurn + e % dim : dim;   // (column dim is not read)
  }

  for (int64_t m0 = (int64_t)blockIdx.x * kNarrowRows; m0 < s.rows; m0 += (int64_t)gridDim.x * kNarrowRows) {
    float xp[4][KS], xw[4][4];   // x as the projections' operand, and [x 1] as dW's
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int k = 0; k < KS; ++k) xp[m][k] = k * 4 + q < dim ? x_at(m0 + m * 16 + l, k * 4 + q) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) xw[m][i] = weights ? x_at(m0 + m * 16 + q * 4 + i, l) : 0.f;
    }
    nv4f dx[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) dx[m] = nv4f{0.f, 0.f, 0.f, 0.f};

    // the next 16 columns' weights, biases and dh, in flight over the products of these
    T next_w[2][EACH];
    Four<T> next_b[2], next_d[4];
    const auto fetch = [&](int b) {
      const int64_t n0 = c0 + b * 16, n = n0 + q * 4;
      const int last = (int)(c1 - n0 < 16 ? c1 - n0 : 16) * dim - 1;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int e = lane + j * 64 < last ? lane + j * 64 : last;   // (every lane loads: no branches)
        next_w[0][j] = ((const T*)a.wg + n0 * dim)[e];
        next_w[1][j] = ((const T*)a.wu + n0 * dim)[e];
      }
      next_b[0].load((const T*)a.bg + n, a.bg ? c1 - n : 0);
      next_b[1].load((const T*)a.bu + n, a.bu ? c1 - n : 0);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int64_t r = m0 + m * 16 + l < s.rows ? m0 + m * 16 + l : s.rows - 1;
        next_d[m].load((const T*)a.dh + r * a.dh_stride + n, n0 + 16 <= c1 ? 4 : c1 - n);
      }
    };
    if (wave < blocks) fetch(wave);
    for (int b = wave; b < blocks; b += kNarrowWaves) {
      const int64_t n0 = c0 + b * 16, n = n0 + q * 4;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < EACH; ++j) {   // (rows past the last hold copies: their columns are masked below)
        wrow[w_to[j]] = to_f(next_w[0][j]);
        wrow[16 * kTurn + w_to[j]] = to_f(next_w[1][j]);
      }
      nv4f bias[2];
      Four<T> dh[4];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[w][i] = next_b[w].at(i);
#pragma unroll
      for (int m = 0; m < 4; ++m) dh[m] = next_d[m];
      if (b + kNarrowWaves < blocks) fetch(b + kNarrowWaves);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      float wp[2][KS], wx[2][4];   // the weights as the projections' operand, and as dx's
#pragma unroll
      for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const float v = wrow[(w * 16 + l) * kTurn + k * 4 + q];
          wp[w][k] = k * 4 + q < dim ? v : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = wrow[(w * 16 + q * 4 + i) * kTurn + l];
          wx[w][i] = n + i < c1 ? v : 0.f;
        }
      }
      nv4f dw[2];
      dw[0] = dw[1] = nv4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        nv4f pg = bias[0], pu = bias[1];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          pg = narrow_mma(wp[0][k], xp[m][k], pg);
          pu = narrow_mma(wp[1][k], xp[m][k], pu);
        }
        const int64_t r = m0 + m * 16 + l;
        float g[4], act[4], slope[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = pg[i], u[i] = pu[i];
        activate<T>(a.act, g, act, slope);
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // (rows and columns that are not there add nothing, also where W is not finite)
          const float d = dh[m].at(i);
          const bool in = r < s.rows && n + i < c1;
          g[i] = in ? d * u[i] * slope[i] : 0.f;
          u[i] = in ? d * act[i] : 0.f;
        }
        if (a.dx)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dx[m] = narrow_mma(wx[0][i], g[i], dx[m]);
            dx[m] = narrow_mma(wx[1][i], u[i], dx[m]);
          }
        if (weights) {
          __builtin_amdgcn_wave_barrier();
          *(nv4f*)(turn + l * kTurn + q * 4) = nv4f{g[0], g[1], g[2], g[3]};
          *(nv4f*)(turn + (16 + l) * kTurn + q * 4) = nv4f{u[0], u[1], u[2], u[3]};
          asm volatile("" ::: "memory");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dw[0] = narrow_mma(xw[m][i], turn[(q * 4 + i) * kTurn + l], dw[0]);
            dw[1] = narrow_mma(xw[m][i], turn[(16 + q * 4 + i) * kTurn + l], dw[1]);
          }
          asm volatile("" ::: "memory");
        }
      }
      const int at = q * 4;
      if (weights && n0 + l < c1 && at < width) {   // row n0 + l of [dW db], four columns a lane
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (gridDim.x > 1) {
            nv4f* to = (nv4f*)(a.dw_parts + ((blockIdx.x * 2 + w) * s.hidden + n0 + l) * width + at);
            *to = m0 == (int64_t)blockIdx.x * kNarrowRows ? dw[w] : *to + dw[w];
          } else {
            T *to = (T*)(w ? a.dwu : a.dwg), *db = (T*)(w ? a.dbu : a.dbg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (at + i < dim && to) to[(n0 + l) * dim + at + i] = from_f<T>(dw[w][i]);
              if (at + i == dim && db) db[n0 + l] = from_f<T>(dw[w][i]);
            }
          }
        }
      }
    }
    if (a.dx) {
      __syncthreads();
      float* mine = lds + wave * kNarrowRows * LD;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(m * 16 + l) * LD + q * 4 + i] = dx[m][i];
      __syncthreads();
      const int left = (int)(s.rows - m0 < kNarrowRows ? s.rows - m0 : kNarrowRows);
      for (int at = threadIdx.x; at < left * dim; at += kNarrowWaves * 64) {
        const float* p = lds + at / dim * LD + at % dim;
        float v = p[0];
#pragma unroll
        for (int w = 1; w < kNarrowWaves; ++w) v += p[w * kNarrowRows * LD];
        if (gridDim.y > 1) {
          a.dx_parts[(blockIdx.y * s.rows + m0) * dim + at] = v;
        } else {
          ((T*)a.dx)[m0 * dim + at] = from_f<T>(v);
        }
      }
      __syncthreads();
    }
  }
}

// Sums of the parts, in order: [dW db] first (`dw_blocks` workgroups), then dx.  Sixteen lanes a value
// where it has that many parts, each a fixed share of them with loads in flight.
template <typename T>
__global__ __launch_bounds__(1024) void k_narrow_join(GatedNarrow a, int64_t groups, int64_t shares, int64_t dw_blocks) {
  __shared__ float sum[16][65];
  const GatedShape s = a.s;
  const int64_t width = NarrowPlan::width(s.dim);
  const bool dw = blockIdx.x < dw_blocks;
  const float* parts = dw ? a.dw_parts : a.dx_parts;
  const int64_t count = dw ? groups : shares, values = dw ? 2 * s.hidden * width : s.rows * s.dim;
  const int64_t block = dw ? blockIdx.x : blockIdx.x - dw_blocks;
  const bool many = count >= 16;
  const int lane = many ? threadIdx.x % 64 : threadIdx.x, part = many ? threadIdx.x / 64 : 0;
  const int64_t c = block * (many ? 64 : 1024) + lane;
  float v = 0.f;
  if (c < values) {
#pragma unroll 8
    for (int64_t p = part; p < count; p += many ? 16 : 1) v += parts[p * values + c];
  }
  if (many) {
    sum[part][lane] = v;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int p = 1; p < 16; ++p) v += sum[p][lane];
  }
  if (c >= values) return;
  if (!dw) {
    ((T*)a.dx)[c] = from_f<T>(v);
    return;
  }
  const int64_t d = c % width, n = c / width % s.hidden;
  const bool up = c >= s.hidden * width;
  T *to = (T*)(up ? a.dwu : a.dwg), *bias = (T*)(up ? a.dbu : a.dbg);
  if (d < s.dim && to) to[n * s.dim + d] = from_f<T>(v);
  if (d == s.dim && bias) bias[n] = from_f<T>(v);
}

// Workgroups along the rows (a part of [dW db] each) and along the columns (a part of dx each), two a CU where the parts
// of neither pass 512 MB: less would cost time where a workgroup adds to its part tile by tile (16000 x
// 8 -> 12288 fp32: 250 parts, 283 MB, 583 us; 57 in 64 MB 752).  Along the rows they are two at
// least: one alone writes dW itself, from one tile of rows.
NarrowPlan gated_narrow_plan(GatedShape s) {
  const int64_t tiles = ceil_div64(s.rows, kNarrowRows), floats = 1 << 27;
  const auto within = [](int64_t n, int64_t least, int64_t most) { return n > most ? most : n < least ? least : n; };
  const int64_t groups = within(within(floats / (2 * s.hidden * NarrowPlan::width(s.dim)), 2, 512), 1, tiles);
  const int64_t most = within(floats / (s.rows * s.dim), 1, ceil_div64(s.hidden, 16 * kNarrowWaves));
  const int64_t cols = ceil_div64(ceil_div64(s.hidden, within(ceil_div64(512, groups), 1, most)), 16) * 16;
  return NarrowPlan{groups, ceil_div64(s.hidden, cols)};
}

template <typename T, int KS>
static void narrow_launch(const GatedNarrow& a, NarrowPlan p, hipStream_t st) {
  k_narrow<T, KS><<<dim3((unsigned)p.groups, (unsigned)p.shares), kNarrowWaves * 64, 0, st>>>(a);
  const auto blocks = [](int64_t values, int64_t count) { return ceil_div64(values, count >= 16 ? 64 : 1024); };
  const bool weights = a.dwg || a.dwu || a.dbg || a.dbu;
  const int64_t dw = weights && p.groups > 1 ? blocks(2 * a.s.hidden * NarrowPlan::width(a.s.dim), p.groups) : 0;
  const int64_t dx = a.dx && p.shares > 1 ? blocks(a.s.rows * a.s.dim, p.shares) : 0;
  if (dw + dx) k_narrow_join<T><<<(unsigned)(dw + dx), 1024, 0, st>>>(a, p.groups, p.shares, dw);
}

template <typename T>
static void narrow_type(const GatedNarrow& a, NarrowPlan p, hipStream_t st) {
  if (a.s.dim <= 4) {
    narrow_launch<T, 1>(a, p, st);
  } else if (a.s.dim <= 8) {
    narrow_launch<T, 2>(a, p, st);
  } else if (a.s.dim <= 12) {
    narrow_launch<T, 3>(a, p, st);
  } else {
    narrow_launch<T, 4>(a, p, st);
  }
}

void gated_narrow(int type, GatedNarrow a, hipStream_t st) {
  const NarrowPlan p = gated_narrow_plan(a.s);
  a.cols = ceil_div64(ceil_div64(a.s.hidden, p.shares), 16) * 16;
  if (type == GSR_F32) {
    narrow_type<float>(a, p, st);
  } else if (type == GSR_BF16) {
    narrow_type<bf16>(a, p, st);
  } else {
    narrow_type<f16>(a, p, st);
  }
}

}  // namespace gsr
