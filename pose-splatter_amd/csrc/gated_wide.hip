// The gated block's products in 16 bits with square tiles of 256 or 128 (wide.h has the layout).
//
//   forward, gradients  a tile is 256 (128) rows by half as many columns of g and the same columns of u
//                       (the first half of its shared memory's rows from Wg, the second from Wu), so
//                       a wave holds both projections of its outputs and the activation joins them
//   dx                  K runs through [dg | du], its other operand through Wg, then Wu
//   dWg, dWu            rows are the columns of [dg | du], K the rows of x
#include "gated_wide.h"

#include "wide.h"

namespace gsr {

template <typename T, int MODE, int SIDE>
__global__ __launch_bounds__(kWideThreads, SIDE == 256 ? 1 : 2) void k_wide(GatedWide a) {
  constexpr bool DUAL = MODE == kWideFwd || MODE == kWideGrad, AKC = MODE != kWideDw, BKC = DUAL;
  constexpr int NB = SIDE / 64, HALF = SIDE / 2, BYTES = SIDE * kWideK * 2;   // blocks a wave and side; its rows
  __shared__ __attribute__((aligned(1024))) char lds[kWideStages][2][BYTES];   // [stage][operand]
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wm = wave % 2, wn = wave / 2;
  const GatedShape s = a.s;
  const int64_t pad = gated_pad(s.hidden);
  int tm, tn;
  wide_tile_of(blockIdx.x, a.mt, a.nt, &tm, &tn);
  const int64_t m0 = (int64_t)tm * SIDE, n0 = (int64_t)tn * (DUAL ? HALF : SIDE);

  // K of this workgroup, and the operands' corners.  Where K is contiguous the descriptor holds the
  // tile's rows of one step; where it runs across rows, a step's rows up to K's end (the last step
  // may be short: `short_bytes`).
  int64_t k0 = 0, k1 = DUAL ? a.kdim : MODE == kWideDx ? 2 * pad : s.rows;
  if constexpr (!DUAL) {
    k0 = blockIdx.z * a.share;
    k1 = k0 + a.share < k1 ? k0 + a.share : k1;
  }
  const int steps = (int)((k1 - k0 + kWideK - 1) / kWideK);
  const auto at = [](const void* p, int64_t i) { return (const char*)p + i * 2; };
  const auto rows_of = [&](int64_t rows, int64_t first, int64_t stride) {   // K contiguous: rows first .. of `rows`
    const int64_t n = rows - first < SIDE ? rows - first : SIDE;
    return n <= 0 ? 0 : ((n - 1) * stride + kWideK) * 2;
  };
  const auto ks_of = [](int64_t n, int64_t stride, int64_t left) {   // K across rows: n K, `left` columns to the row's end
    return n <= 0 ? 0 : ((n < kWideK ? n : kWideK) - 1) * stride * 2 + left * 2;
  };
  WideSource sa, sb, sb2;
  uint32_t a_step, b_step, a_short = 0, b_short = 0;
  int64_t a_stride, b_stride;
  int shorts = steps, turn = -1;   // steps from `shorts` on are short; at step `turn` the second matrix begins
  if constexpr (DUAL) {
    a_stride = a.x_stride, b_stride = a.w_stride;
    sa = WideSource(at(a.x, m0 * a_stride), rows_of(s.rows, m0, a_stride));
    const int64_t n = s.hidden - n0 < HALF ? s.hidden - n0 : HALF, bytes = n <= 0 ? 0 : ((n - 1) * b_stride + kWideK) * 2;
    sb = WideSource(at(a.wg, n0 * b_stride), bytes);
    sb2 = WideSource(at(a.wu, n0 * b_stride), bytes);
    a_step = b_step = kWideK * 2;
  } else if constexpr (MODE == kWideDx) {
    a_stride = 2 * pad, b_stride = a.w_stride;
    sa = WideSource(at(a.dgu, m0 * a_stride + k0), rows_of(s.rows, m0, a_stride));
    // K rows of Wg, then of Wu, each followed by up to pad - hidden < 64 rows of nothing
    const int64_t kw = k0 < pad ? k0 : k0 - pad;   // (pad is whole steps: none straddles the matrices)
    sb = WideSource(at(k0 < pad ? a.wg : a.wu, kw * b_stride + n0), ks_of(kWideK, b_stride, a.kdim - n0));
    sb2 = WideSource(at(a.wu, n0), 0);
    a_step = kWideK * 2, b_step = (uint32_t)(kWideK * b_stride * 2);
    turn = k0 < pad ? (int)((pad - k0) / kWideK) : -1;
  } else {
    a_stride = 2 * pad, b_stride = a.x_stride;
    sa = WideSource(at(a.dgu, k0 * a_stride + m0), ks_of(k1 - k0, a_stride, a_stride - m0));
    sb = WideSource(at(a.x, k0 * b_stride + n0), ks_of(k1 - k0, b_stride, a.kdim - n0));
    a_step = (uint32_t)(kWideK * a_stride * 2), b_step = (uint32_t)(kWideK * b_stride * 2);
    a_short = (uint32_t)ks_of((k1 - k0) % kWideK, a_stride, a_stride - m0);
    b_short = (uint32_t)ks_of((k1 - k0) % kWideK, b_stride, a.kdim - n0);
    shorts = (int)((k1 - k0) / kWideK);
  }
  WideTile<AKC, SIDE> ta;
  WideTile<BKC, SIDE> tb;
  ta.init(a_stride * 2, wm * HALF);
  tb.init(b_stride * 2, DUAL ? wn * (HALF / 2) : wn * HALF);

  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0][0] + wave * 1024);
  int next = 0;   // the next step to load
  v4i da, db, db2;
  const auto begin = [&]() {   // (a step past K's end is nothing: descriptors of no length)
    if constexpr (MODE == kWideDx) {
      if (next == turn) sb.lo = sb2.lo, sb.hi = sb2.hi;
      // the rows left of this matrix
      const int64_t k = k0 + (int64_t)next * kWideK, n = s.hidden - (k < pad ? k : k - pad);
      sb.bytes = (uint32_t)ks_of(n, b_stride, a.kdim - n0);
    }
    if constexpr (MODE == kWideDw) {
      if (next == shorts) sa.bytes = a_short, sb.bytes = b_short;
    }
    da = sa.descriptor(next < steps);
    db = sb.descriptor(next < steps);
    if constexpr (DUAL) db2 = sb2.descriptor(next < steps);
    sa.advance(a_step);
    sb.advance(b_step);
    if constexpr (DUAL) sb2.advance(b_step);
    ++next;
  };
  constexpr int LOADS = BYTES / 4096;
  const auto load = [&](int i, uint32_t to) {   // one of 2 LOADS into the stage at `to`
    if (i < LOADS) {
      wide_load(da, ta.at[i % LOADS], to, i * 4096);
    } else if (DUAL && i >= LOADS * 3 / 2) {
      wide_load(db2, tb.at[i - LOADS * 3 / 2], to, i * 4096);
    } else {
      wide_load(db, tb.at[i - LOADS], to, i * 4096);
    }
  };

  v16f acc[NB][NB];   // [n block][m block]
#pragma unroll
  for (int i = 0; i < NB * NB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i / NB][i % NB][j] = 0.f;
  v8s fa[2][NB], fb[2][NB];
  const char* base = &lds[0][0][0];
  const auto operand = [&](int stage, int kk, int i) {   // one of 2 NB
    const char* p = base + stage * 2 * BYTES;
    if (i < NB) {
      fa[kk][i % NB] = ta.operand(p, i * 32, kk);
    } else {
      const int b = i % NB;
      fb[kk][b] = tb.operand(p + BYTES, DUAL && b >= NB / 2 ? HALF + (b - NB / 2) * 32 : b * 32, kk);
    }
  };
  // Half a step: the products of kk, and between them the reads of the next half's operands, then half
  // of a stage's loads.  One wave a SIMD issues all of it, so every other instruction sits in a
  // product's shadow (32 cycles, six or so instructions); the order is as written.
  const auto half_step = [&](int kk, int from, uint32_t to) {
#pragma unroll
    for (int i = 0; i < NB * NB; ++i) {
      acc[i / NB][i % NB] = wide_mma<T>(fb[kk][i / NB], fa[kk][i % NB], acc[i / NB][i % NB]);
      constexpr int EVERY = NB * NB / LOADS, READS = 4 / NB;   // reads a product: 1 of 16, 2 of 4
#pragma unroll
      for (int j = 0; j < READS; ++j)
        if (i * READS + j < 2 * NB) operand(from, kk ^ 1, i * READS + j);
      if (i % EVERY == EVERY - 1) load(kk * LOADS + i / EVERY, to);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int AHEAD = kWideStages - 1, FLIGHT = (AHEAD - 2) * 2 * LOADS + LOADS;
#pragma unroll
  for (int b = 0; b < AHEAD; ++b) {
    begin();
#pragma unroll
    for (int i = 0; i < 2 * LOADS; ++i) load(i, lds0 + b * 2 * BYTES);
  }
  wide_wait<(AHEAD - 1) * 2 * LOADS>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) operand(0, 0, i);
  int stage = 0;
  for (int st = 0; st < steps; ++st) {
    const int after = stage == AHEAD ? 0 : stage + 1;
    const uint32_t to = lds0 + (stage == 0 ? AHEAD : stage - 1) * 2 * BYTES;   // the step before's stage: read by all
    begin();
    half_step(0, stage, to);
    // This stage's last operands are in registers, and the next stage has landed: for every wave,
    // after the barrier.
    wide_wait<FLIGHT>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    half_step(1, after, to);
    stage = after;
  }

  // Each wave passes its sums, 32 rows of a block row at a time, through its own part of the shared memory
  // (no wave reads a tile any more after the barrier): there a lane takes eight neighbouring columns,
  // so that rows are read and written in whole lines.
  wide_wait<0>();   // (the loads past K's end write zeros)
  __syncthreads();
  constexpr int LD = HALF + 4;   // floats a row: a wave's columns and 4 to spread the banks
  static_assert(4 * 32 * LD * sizeof(float) <= sizeof(lds), "the waves' rows fit the tiles' memory");
  float* mine = (float*)&lds[0][0][0] + wave * 32 * LD;
  constexpr int COLS = DUAL ? HALF / 2 : HALF, LANES = COLS / 8, ROWS = 64 / LANES;   // lanes a row, rows a pass
  const int c = lane % LANES * 8;
  const int64_t n = n0 + wn * COLS + c, left_n = (DUAL ? s.hidden : s.dim) - n;
  float gb[8] = {}, ub[8] = {}, sg[8] = {}, su[8] = {};
  if constexpr (DUAL) {
    load_upto((const T*)a.bg + n, a.bg ? left_n : 0, gb);
    load_upto((const T*)a.bu + n, a.bu ? left_n : 0, ub);
  }
#pragma unroll
  for (int mb = 0; mb < NB; ++mb) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)   // a lane holds row lane % 32, columns 8 q + 4 (lane / 32) + 0..3 of a block
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(v4f*)(mine + lane % 32 * LD + nb * 32 + q * 8 + lane / 32 * 4) =
            v4f{acc[nb][mb][q * 4], acc[nb][mb][q * 4 + 1], acc[nb][mb][q * 4 + 2], acc[nb][mb][q * 4 + 3]};
    wide_fence();
    const int64_t first = m0 + wm * HALF + mb * 32;
#pragma unroll 1
    for (int r = lane / LANES; r < 32; r += ROWS) {
      const int64_t m = first + r;
      if (m >= (MODE == kWideDw ? 2 * pad : s.rows)) break;
      float g[8], u[8], d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[i] = mine[r * LD + c + i];
        if constexpr (DUAL) u[i] = mine[r * LD + COLS + c + i];
      }
      if constexpr (DUAL) {
        if constexpr (MODE == kWideGrad) load_upto((const T*)a.dh + m * a.dh_stride + n, left_n, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float act, slope;
          g[i] += gb[i];
          u[i] += ub[i];
          activate<T>(a.act, g[i], act, slope);
          if constexpr (MODE == kWideFwd) {
            g[i] = act * u[i];
          } else {
            g[i] = i < left_n ? d[i] * u[i] * slope : 0.f;   // (the padding holds zeros)
            u[i] = i < left_n ? d[i] * act : 0.f;
            sg[i] += g[i];
            su[i] += u[i];
          }
        }
      }
      if constexpr (MODE == kWideFwd) {
        store_upto((T*)a.h + m * s.hidden + n, left_n, g);
      } else if constexpr (MODE == kWideGrad) {
        if (n < pad) {
          store_vec((T*)a.dgu + m * 2 * pad + n, g);
          store_vec((T*)a.dgu + m * 2 * pad + pad + n, u);
        }
      } else if constexpr (MODE == kWideDx) {
        if (a.parts) {
          store_upto(a.parts + (blockIdx.z * s.rows + m) * s.dim + n, left_n, g);
        } else {
          store_upto((T*)a.dx + m * s.dim + n, left_n, g);
        }
      } else {
        const int which = m >= pad;
        const int64_t row = m - which * pad;
        if (row < s.hidden) {
          if (a.parts) {
            store_upto(a.parts + ((blockIdx.z * 2 + which) * s.hidden + row) * s.dim + n, left_n, g);
          } else if (T* to = (T*)(which ? a.dwu : a.dwg)) {
            store_upto(to + row * s.dim + n, left_n, g);
          }
        }
      }
    }
    wide_fence();
  }
  if (MODE == kWideGrad && a.parts) {   // column sums of the wave's rows
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int d = LANES; d < 64; d <<= 1) {
        sg[i] += __shfl_xor(sg[i], d);
        su[i] += __shfl_xor(su[i], d);
      }
      if (lane < LANES && i < left_n) {
        float* to = a.parts + (int64_t)(tm * 2 + wm) * 2 * s.hidden + n + i;
        to[0] = sg[i];
        to[s.hidden] = su[i];
      }
    }
  }
}

template <typename T, int SIDE>
static void wide_launch(int mode, const GatedWide& a, int shares, hipStream_t st) {
  const dim3 grid((unsigned)(a.mt * a.nt), 1, (unsigned)shares);
  if (mode == kWideFwd) {
    k_wide<T, kWideFwd, SIDE><<<grid, kWideThreads, 0, st>>>(a);
  } else if (mode == kWideGrad) {
    k_wide<T, kWideGrad, SIDE><<<grid, kWideThreads, 0, st>>>(a);
  } else if (mode == kWideDx) {
    k_wide<T, kWideDx, SIDE><<<grid, kWideThreads, 0, st>>>(a);
  } else {
    k_wide<T, kWideDw, SIDE><<<grid, kWideThreads, 0, st>>>(a);
  }
}

void gated_wide(int type, int mode, int side, GatedWide a, int shares, hipStream_t st) {
  const int64_t pad = gated_pad(a.s.hidden);
  a.mt = ceil_div(mode == kWideDw ? 2 * pad : a.s.rows, side);
  a.nt = mode <= kWideGrad ? ceil_div(pad, side / 2) : ceil_div(a.s.dim, side);
  if (type == GSR_BF16 && side == 256) {
    wide_launch<bf16, 256>(mode, a, shares, st);
  } else if (type == GSR_BF16) {
    wide_launch<bf16, 128>(mode, a, shares, st);
  } else if (side == 256) {
    wide_launch<f16, 256>(mode, a, shares, st);
  } else {
    wide_launch<f16, 128>(mode, a, shares, st);
  }
}

}  // namespace gsr
