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
  __shared__ __attribute__((aligned(1024))) char lds[2][2][BYTES];   // [buffer][operand]
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wm = wave % 2, wn = wave / 2;
  const GatedShape s = a.s;
  const int64_t pad = gated_pad(s.hidden);
  int tm, tn;
  wide_tile_of(blockIdx.x, a.mt, a.nt, &tm, &tn);
  const int64_t m0 = (int64_t)tm * SIDE, n0 = (int64_t)tn * (DUAL ? HALF : SIDE);

  // K of this workgroup, and the operands' first bytes
  int64_t k0 = 0, k1 = DUAL ? a.kdim : MODE == kWideDx ? 2 * pad : s.rows;
  if constexpr (!DUAL) {
    k0 = blockIdx.z * a.share;
    k1 = k0 + a.share < k1 ? k0 + a.share : k1;
  }
  const int steps = (int)((k1 - k0 + kWideK - 1) / kWideK);
  WideSource sa, sb, sb2;
  int64_t a_step, b_step, a_stride, b_stride;
  const auto from = [](const void* p, int64_t at, int64_t end) { return WideSource{(const char*)p + at * 2, (end - at) * 2}; };
  if constexpr (DUAL) {
    a_stride = a.x_stride, b_stride = a.w_stride;
    sa = from(a.x, m0 * a_stride, (s.rows - 1) * a_stride + a.kdim);
    sb = from(a.wg, n0 * b_stride, (s.hidden - 1) * b_stride + a.kdim);
    sb2 = from(a.wu, n0 * b_stride, (s.hidden - 1) * b_stride + a.kdim);
    a_step = b_step = kWideK * 2;
  } else if constexpr (MODE == kWideDx) {
    a_stride = 2 * pad, b_stride = a.w_stride;
    sa = from(a.dgu, m0 * a_stride + k0, s.rows * a_stride);
    const int64_t kw = k0 < pad ? k0 : k0 - pad;   // (pad is whole steps: none straddles Wg and Wu)
    sb = from(k0 < pad ? a.wg : a.wu, kw * b_stride + n0, (s.hidden - 1) * b_stride + a.kdim);
    sb2 = from(a.wu, n0, (s.hidden - 1) * b_stride + a.kdim);
    a_step = kWideK * 2, b_step = kWideK * b_stride * 2;
  } else {
    a_stride = 2 * pad, b_stride = a.x_stride;
    sa = from(a.dgu, k0 * a_stride + m0, k1 * a_stride);
    sb = from(a.x, k0 * b_stride + n0, (k1 - 1) * b_stride + a.kdim);
    a_step = kWideK * a_stride * 2, b_step = kWideK * b_stride * 2;
  }
  WideTile<AKC, SIDE> ta;
  WideTile<BKC, SIDE> tb;
  ta.init(a_stride * 2, wm * HALF);
  tb.init(b_stride * 2, DUAL ? wn * (HALF / 2) : wn * HALF);

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0][0];
  int64_t left = k1 - k0;   // K left at the next tile's start
  int next = 0;             // the next tile to load
  v4i da, db, db2;
  const auto begin = [&]() {   // (a tile past K's end is nothing: descriptors of no length)
    da = sa.descriptor(next < steps);
    db = sb.descriptor(next < steps);
    if constexpr (DUAL) db2 = sb2.descriptor(next < steps);
  };
  constexpr int LOADS = SIDE / 32;
  const auto load = [&](int i, int buf) {   // one of 2 LOADS
    const uint32_t to = lds0 + buf * 2 * BYTES;
    if (i < LOADS) {
      ta.load(da, to, i, i, left);
    } else if (DUAL && i >= LOADS * 3 / 2) {
      tb.load(db2, to + BYTES, i - LOADS, i - LOADS * 3 / 2, left);
    } else {
      tb.load(db, to + BYTES, i - LOADS, i - LOADS, left);
    }
  };
  const auto end = [&]() {
    sa.advance(a_step);
    sb.advance(b_step);
    if constexpr (DUAL) sb2.advance(b_step);
    left -= kWideK;
    ++next;
    if constexpr (MODE == kWideDx)
      if (k0 + (int64_t)next * kWideK == pad) sb = sb2;
  };

  v16f acc[NB][NB];   // [n block][m block]
#pragma unroll
  for (int i = 0; i < NB * NB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i / NB][i % NB][j] = 0.f;
  v8s fa[2][NB], fb[2][NB];
  const auto operands = [&](int buf, int kk, int set) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      fa[set][b] = ta.operand(lds[buf][0], b * 32, kk);
      fb[set][b] = tb.operand(lds[buf][1], DUAL && b >= NB / 2 ? HALF + (b - NB / 2) * 32 : b * 32, kk);
    }
  };
  const auto mma = [&](int set, int i) {
    acc[i / NB][i % NB] = wide_mma<T>(fb[set][i / NB], fa[set][i % NB], acc[i / NB][i % NB]);
  };

#pragma unroll
  for (int b = 0; b < 2; ++b) {
    begin();
#pragma unroll
    for (int i = 0; i < 2 * LOADS; ++i) load(i, b);
    end();
  }
  wide_wait();
  __syncthreads();
  operands(0, 0, 0);
  for (int st = 0; st < steps; ++st) {
    const int buf = st & 1;
#pragma unroll
    for (int kk = 0; kk < 3; ++kk) {
      operands(buf, kk + 1, (kk + 1) & 1);   // in flight over the products (the scheduler would sink them)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NB * NB; ++i) mma(kk & 1, i);
    }
    // The last operands of this buffer are in registers and the next buffer's loads, a step old,
    // have landed: for every wave, after the barrier.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    operands(buf ^ 1, 0, 0);
    begin();
#pragma unroll
    for (int i = 0; i < NB * NB; ++i) {   // loads between the products, rather than all in a row
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2 * LOADS / (NB * NB); ++j) load(i * (2 * LOADS / (NB * NB)) + j, buf);
      mma(1, i);
    }
    end();
  }

  // Each wave passes its sums, 32 rows of a block row at a time, through its own part of the shared memory
  // (no wave reads a tile any more after the barrier): there a lane takes eight neighbouring columns,
  // so that rows are read and written in whole lines.
  wide_wait();   // (the loads past K's end write zeros)
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
