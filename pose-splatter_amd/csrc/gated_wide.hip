// The gated block's products with square tiles of 256 (16 bits) or 128 (wide.h has the layout).
//
//   forward, gradients  a tile is 256 (128) rows by half as many columns of g and the same columns of u
//                       (the first half of its shared memory's rows from Wg, the second from Wu), so
//                       a wave holds both projections of its outputs and the activation joins them
//   dx                  K runs through [dg | du], its other operand through Wg, then Wu
//   dWg, dWu            rows are the columns of [dg | du], K the rows of x
//
// Averages of 60 passes (the quickest in brackets), 16384 x 2048 -> 5632 bf16: forward 682 us (652; 1110
// TFLOP/s, writing its kept projections as well), dx 581 (559; 1300), dW 603 (572; 1250); 16000 x
// 256 -> 512 fp32 90 us (85), and dx and dW side by side 149 (140): 93 and 113 of the card's 153
// TFLOP/s in fp32.  Those are one or two rounds of tiles whose first loads and last stores nothing
// hides; the epilogue leaves two of the ring's five slots (three of them at 256) to the next tile's
// first loads, which are not issued there.
#include "gated_wide.h"

#include "wide.h"

namespace gsr {

// Eight neighbouring results of dx, or of the weight gradients, whose rows are [dg | pad | du | pad]'s columns.
template <typename T, int MODE>
__device__ __forceinline__ void wide_store(const GatedWide& a, int64_t m, int64_t n, const float (&v)[8]) {
  const GatedShape s = a.s;
  if constexpr (MODE == kWideDx) {
    if (m < s.rows) store_upto((T*)a.dx + m * s.dim + n, s.dim - n, v);
  } else {
    const int64_t pad = gated_pad(s.hidden);
    const int which = m >= pad;
    const int64_t row = m - which * pad;
    T* to = (T*)(which ? a.dwu : a.dwg);
    if (row < s.hidden && to) store_upto(to + row * s.dim + n, s.dim - n, v);
  }
}

template <int N>
struct Count {
  static constexpr int value = N;
};

// Workgroup `id` of a product; lds: kWideSlots operand tiles.
template <typename T, int MODE, int SIDE>
__device__ __forceinline__ void wide_product(const GatedWide& a, int id, char (*lds)[SIDE * 128]) {
  constexpr bool DUAL = MODE == kWideFwd || MODE == kWideGrad, AKC = MODE != kWideDw, BKC = DUAL;
  constexpr int NB = SIDE / 64, HALF = SIDE / 2, BYTES = SIDE * 128;   // blocks a wave and side; its rows
  constexpr int ES = sizeof(T), K = kWideK<T>;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wm = wave % 2, wn = wave / 2;
  const GatedShape s = a.s;
  const int64_t pad = gated_pad(s.hidden);
  // Whole tiles first; those that would leave CUs idle in the last round are cut into shares of K.
  int tm, tn, share = -1;
  if constexpr (MODE != kWideGrad) {
    if (id >= a.whole) {
      share = (id - a.whole) / a.cut;
      id = a.whole + (id - a.whole) % a.cut;
    }
  }
  wide_tile_of(id, a.mt, a.nt, &tm, &tn);
  const int64_t m0 = (int64_t)tm * SIDE, n0 = (int64_t)tn * (DUAL ? HALF : SIDE);

  // K of this workgroup, and the operands' corners.  Where K is contiguous the descriptor holds the
  // tile's rows of one step; where it runs across rows, a step's rows up to K's end (the last step
  // may be short: `short_bytes`).
  int64_t k0 = 0, k1 = DUAL ? a.kdim : MODE == kWideDx ? 2 * pad : s.rows;
  if constexpr (MODE != kWideGrad) {
    if (share >= 0) {
      const int64_t all = (k1 + K - 1) / K;
      k0 = all * share / a.shares * K;
      if (share + 1 < a.shares) k1 = all * (share + 1) / a.shares * K;
    }
  }
  const int steps = (int)((k1 - k0 + K - 1) / K);
  const auto at = [](const void* p, int64_t i) { return (const char*)p + i * ES; };
  const auto rows_of = [&](int64_t rows, int64_t first, int64_t stride) {   // K contiguous: rows first .. of `rows`
    const int64_t n = rows - first < SIDE ? rows - first : SIDE;
    return n <= 0 ? 0 : ((n - 1) * stride + K) * ES;
  };
  const auto ks_of = [](int64_t n, int64_t stride, int64_t left) {   // K across rows: n K, `left` columns to the row's end
    return n <= 0 ? 0 : ((n < K ? n : K) - 1) * stride * ES + left * ES;
  };
  WideSource sa, sb, sb2;
  uint32_t a_step, b_step, a_short = 0, b_short = 0;
  int64_t a_stride, b_stride;
  int shorts = steps, turn = -1;   // steps from `shorts` on are short; at step `turn` the second matrix begins
  if constexpr (DUAL) {
    a_stride = a.x_stride, b_stride = a.w_stride;
    sa = WideSource(at(a.x, m0 * a_stride + k0), rows_of(s.rows, m0, a_stride));
    const int64_t n = s.hidden - n0 < HALF ? s.hidden - n0 : HALF, bytes = n <= 0 ? 0 : ((n - 1) * b_stride + K) * ES;
    sb = WideSource(at(a.wg, n0 * b_stride + k0), bytes);
    sb2 = WideSource(at(a.wu, n0 * b_stride + k0), bytes);
    a_step = b_step = K * ES;
  } else if constexpr (MODE == kWideDx) {
    a_stride = 2 * pad, b_stride = a.w_stride;
    sa = WideSource(at(a.dgu, m0 * a_stride + k0), rows_of(s.rows, m0, a_stride));
    // K rows of Wg, then of Wu, each followed by up to pad - hidden < 64 rows of nothing
    const int64_t kw = k0 < pad ? k0 : k0 - pad;   // (pad is whole steps: none straddles the matrices)
    sb = WideSource(at(k0 < pad ? a.wg : a.wu, kw * b_stride + n0), ks_of(K, b_stride, a.kdim - n0));
    sb2 = WideSource(at(a.wu, n0), 0);
    a_step = K * ES, b_step = (uint32_t)(K * b_stride * ES);
    turn = k0 < pad ? (int)((pad - k0) / K) : -1;
  } else {
    a_stride = 2 * pad, b_stride = a.x_stride;
    sa = WideSource(at(a.dgu, k0 * a_stride + m0), ks_of(k1 - k0, a_stride, a_stride - m0));
    sb = WideSource(at(a.x, k0 * b_stride + n0), ks_of(k1 - k0, b_stride, a.kdim - n0));
    a_step = (uint32_t)(K * a_stride * ES), b_step = (uint32_t)(K * b_stride * ES);
    a_short = (uint32_t)ks_of((k1 - k0) % K, a_stride, a_stride - m0);
    b_short = (uint32_t)ks_of((k1 - k0) % K, b_stride, a.kdim - n0);
    shorts = (int)((k1 - k0) / K);
  }
  WideTile<T, AKC, SIDE> ta;
  WideTile<T, BKC, SIDE> tb;
  ta.init(a_stride * ES, wm * HALF);
  tb.init(b_stride * ES, DUAL ? wn * (HALF / 2) : wn * HALF);

  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0] + wave * 1024);
  // A step's operand tiles are loaded one after the other, A then B; next_*: the step whose tile is next.
  // (A step past K's end is nothing: descriptors of no length.)
  int next_a = 0, next_b = 0, left_a = (int)(k1 - k0), left_b = left_a;
  v4i da, db, db2;
  const auto begin_a = [&]() {
    if constexpr (MODE == kWideDw)
      if (next_a == shorts) sa.bytes = a_short;
    da = sa.descriptor(next_a < steps);
    sa.advance(a_step);
    left_a = (int)(k1 - k0) - next_a * K;
    ++next_a;
  };
  const auto begin_b = [&]() {
    if constexpr (MODE == kWideDx) {
      if (next_b == turn) sb.lo = sb2.lo, sb.hi = sb2.hi;
      const int64_t k = k0 + (int64_t)next_b * K, n = s.hidden - (k < pad ? k : k - pad);   // rows left in the matrix
      sb.bytes = (uint32_t)ks_of(n, b_stride, a.kdim - n0);
    }
    if constexpr (MODE == kWideDw)
      if (next_b == shorts) sb.bytes = b_short;
    db = sb.descriptor(next_b < steps);
    if constexpr (DUAL) db2 = sb2.descriptor(next_b < steps);
    sb.advance(b_step);
    if constexpr (DUAL) sb2.advance(b_step);
    left_b = (int)(k1 - k0) - next_b * K;
    ++next_b;
  };
  constexpr int LOADS = BYTES / 4096;
  const auto load_a = [&](int i, int slot) { wide_load(da, ta.offset(i, left_a), lds0 + slot * BYTES, i * 4096); };
  const auto load_b = [&](int i, int slot) {
    if (DUAL && i >= LOADS / 2) {
      wide_load(db2, tb.offset(i - LOADS / 2, left_b), lds0 + slot * BYTES, i * 4096);
    } else {
      wide_load(db, tb.offset(i, left_b), lds0 + slot * BYTES, i * 4096);
    }
  };

  v16f acc[NB][NB];   // [n block][m block]
#pragma unroll
  for (int i = 0; i < NB * NB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i / NB][i % NB][j] = 0.f;
  v8s fa[2][NB], fb[2][NB];
  const auto operand = [&](int slot_a, int slot_b, int kk, int i) {   // one of 2 NB
    if (i < NB) {
      fa[kk & 1][i % NB] = ta.operand(&lds[slot_a][0], i * 32, kk);
    } else {
      const int b = i % NB;
      fb[kk & 1][b] = tb.operand(&lds[slot_b][0], DUAL && b >= NB / 2 ? HALF + (b - NB / 2) * 32 : b * 32, kk);
    }
  };
  // A quarter of a step: its products, and between them the reads of the next quarter's operands
  // (of kk `read` in the slots given), then `loads` of the LOADS loads that `load` issues.  One wave a
  // SIMD issues all of it, so every other instruction sits in a product's shadow (32 cycles, six
  // or so instructions); the order is as written.
  const auto quarter = [&](int kk, int slot_a, int slot_b, int read, auto loads, auto load) {
#pragma unroll
    for (int i = 0; i < NB * NB; ++i) {
      acc[i / NB][i % NB] = wide_mma<T>(fb[kk & 1][i / NB], fa[kk & 1][i % NB], acc[i / NB][i % NB]);
      constexpr int READS = 4 / NB;   // reads a product: 1 of 16, 2 of 4
#pragma unroll
      for (int j = 0; j < READS; ++j)
        if (i * READS + j < 2 * NB) operand(slot_a, slot_b, read, i * READS + j);
      constexpr int N = decltype(loads)::value;
      if constexpr (N > 0) {
        constexpr int EVERY = NB * NB / N;
        if (i % EVERY == EVERY - 1) load(i / EVERY);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto nothing = [](int) {};

#pragma unroll
  for (int b = 0; b < 2; ++b) {
    begin_a();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_a(i, 2 * b);
    begin_b();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_b(i, 2 * b + 1);
  }
  wide_wait<2 * LOADS>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) operand(0, 1, 0, i);
  const auto plus = [](int slot, int n) { return slot + n < kWideSlots ? slot + n : slot + n - kWideSlots; };
  int slot_a = 0, slot_b = 1;   // of this step; the next step's are two on, the one after's four
  for (int st = 0; st < steps; ++st) {
    const int into_a = plus(slot_a, 4), next_slot_a = plus(slot_a, 2), next_slot_b = plus(slot_b, 2);
    begin_a();   // A of the step after the next, into the slot of B of the step before
    quarter(0, slot_a, slot_b, 1, Count<LOADS / 2>{}, [&](int i) { load_a(i, into_a); });
    quarter(1, slot_a, slot_b, 2, Count<LOADS / 2>{}, [&](int i) { load_a(LOADS / 2 + i, into_a); });
    quarter(2, slot_a, slot_b, 3, Count<0>{}, nothing);
    // This step's last operands are in registers and the next step's tiles have landed (only the A
    // above may be in flight): for every wave, after the barrier.
    wide_wait<LOADS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    begin_b();   // B of the step after the next, into this step's slot of A
    quarter(3, next_slot_a, next_slot_b, 0, Count<LOADS>{}, [&](int i) { load_b(i, slot_a); });
    slot_a = next_slot_a;
    slot_b = next_slot_b;
  }

  // Each wave passes its sums, 32 rows of a block row at a time, through its own part of the shared memory
  // (no wave reads a tile any more after the barrier): there a lane takes eight neighbouring columns,
  // so that rows are read and written in whole lines.
  wide_wait<0>();   // (the loads past K's end write zeros)
  __syncthreads();
  constexpr int LD = HALF + 4;   // floats a row: a wave's columns and 4 to spread the banks
  static_assert(4 * 32 * LD * sizeof(float) <= kWideSlots * BYTES, "the waves' rows fit the tiles' memory");
  float* mine = (float*)&lds[0][0] + wave * 32 * LD;
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
      float g[8], u[8], d[8];
      if constexpr (MODE == kWideGrad) load_upto((const T*)a.dh + m * a.dh_stride + n, m < s.rows ? left_n : 0, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[i] = mine[r * LD + c + i];
        if constexpr (DUAL) u[i] = mine[r * LD + COLS + c + i];
      }
      if constexpr (DUAL) {
        if (m >= s.rows) continue;
        if (MODE == kWideFwd && share >= 0) {   // for wide_join_fwd
          float* to = a.cuts + ((int64_t)share * a.cut + (id - a.whole)) * SIDE * SIDE + (m - m0) * SIDE + wn * COLS + c;
          store_vec(to, g);
          store_vec(to + HALF, u);
          continue;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          g[i] += gb[i];
          u[i] += ub[i];
        }
        if constexpr (MODE == kWideFwd)
          if (a.kept && n < pad) Kept<T>(a.kept, s.rows, s.hidden).store(m * pad + n, g, u);
        float act[8], slope[8];
        activate<T>(a.act, g, act, slope);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (MODE == kWideFwd) {
            g[i] = act[i] * u[i];
          } else {
            g[i] = i < left_n ? d[i] * u[i] * slope[i] : 0.f;   // (the padding holds zeros)
            u[i] = i < left_n ? d[i] * act[i] : 0.f;
            sg[i] += g[i];
            su[i] += u[i];
          }
        }
      }
      if constexpr (MODE == kWideFwd) {
        store_upto((T*)a.h + m * s.hidden + n, left_n, g);
      } else if constexpr (MODE == kWideGrad) {
        if (n < pad && a.dgu32) {
          store_vec((float*)a.dgu + m * 2 * pad + n, g);
          store_vec((float*)a.dgu + m * 2 * pad + pad + n, u);
        } else if (n < pad) {
          store_vec((T*)a.dgu + m * 2 * pad + n, g);
          store_vec((T*)a.dgu + m * 2 * pad + pad + n, u);
        }
      } else if (share >= 0) {   // the whole tile, for wide_join
        float* to = a.cuts + ((int64_t)share * a.cut + (id - a.whole)) * SIDE * SIDE;
        store_vec(to + (m - m0) * SIDE + wn * COLS + c, g);
      } else {
        wide_store<T, MODE>(a, m, n, g);
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

template <typename T, int MODE, int SIDE>
__global__ __launch_bounds__(kWideThreads, SIDE == 256 ? 1 : 2) void k_wide(GatedWide a) {
  __shared__ __attribute__((aligned(1024))) char lds[kWideSlots][SIDE * 128];
  wide_product<T, MODE, SIDE>(a, blockIdx.x, lds);
}

// dx by the first `split` workgroups and the weight gradients by the others, side by side: neither alone fills
// the card to its end.
template <typename T>
__global__ __launch_bounds__(kWideThreads, 2) void k_wide_back(GatedWide x, GatedWide w, int split) {
  __shared__ __attribute__((aligned(1024))) char lds[kWideSlots][128 * 128];
  if ((int)blockIdx.x < split) {
    wide_product<T, kWideDx, 128>(x, blockIdx.x, lds);
  } else {
    wide_product<T, kWideDw, 128>(w, blockIdx.x - split, lds);
  }
}

// The cut tiles' results: the sums of their shares, in order.
template <typename T, int MODE, int SIDE>
__device__ __forceinline__ void wide_join(const GatedWide& a, int block) {
  constexpr int EACH = SIDE * SIDE / 8 / 256;   // workgroups a tile
  const int tile = block / EACH, at = (block % EACH * 256 + threadIdx.x) * 8;
  int tm, tn;
  wide_tile_of(a.whole + tile, a.mt, a.nt, &tm, &tn);
  const float* p = a.cuts + (int64_t)tile * SIDE * SIDE + at;
  const int64_t each = (int64_t)a.cut * SIDE * SIDE;
  float v[8] = {};
#pragma unroll 4
  for (int i = 0; i < a.shares; ++i) {
    float w[8];
    load_vec(p + i * each, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += w[j];
  }
  wide_store<T, MODE>(a, (int64_t)tm * SIDE + at / SIDE, (int64_t)tn * SIDE + at % SIDE, v);
}

template <typename T, int MODE, int SIDE>
__global__ __launch_bounds__(256) void k_wide_join(GatedWide a) { wide_join<T, MODE, SIDE>(a, blockIdx.x); }

template <typename T>
__global__ __launch_bounds__(256) void k_wide_join_back(GatedWide x, GatedWide w, int split) {
  if ((int)blockIdx.x < split) {
    wide_join<T, kWideDx, 128>(x, blockIdx.x);
  } else {
    wide_join<T, kWideDw, 128>(w, blockIdx.x - split);
  }
}

// The forward's: both projections' sums, and from them the outputs.
template <typename T, int SIDE>
__global__ __launch_bounds__(256) void k_wide_join_fwd(GatedWide a) {
  constexpr int HALF = SIDE / 2, EACH = SIDE * HALF / 8 / 256;
  const GatedShape s = a.s;
  const int tile = blockIdx.x / EACH, at = (blockIdx.x % EACH * 256 + threadIdx.x) * 8;
  int tm, tn;
  wide_tile_of(a.whole + tile, a.mt, a.nt, &tm, &tn);
  const int64_t m = (int64_t)tm * SIDE + at / HALF, n = (int64_t)tn * HALF + at % HALF, pad = gated_pad(s.hidden);
  if (m >= s.rows || n >= pad) return;
  const float* p = a.cuts + (int64_t)tile * SIDE * SIDE + at / HALF * SIDE + at % HALF;
  const int64_t each = (int64_t)a.cut * SIDE * SIDE, left = s.hidden - n;
  float g[8], u[8], act[8], slope[8];
  load_upto((const T*)a.bg + n, a.bg ? left : 0, g);
  load_upto((const T*)a.bu + n, a.bu ? left : 0, u);
#pragma unroll 4
  for (int i = 0; i < a.shares; ++i) {
    float v[8], w[8];
    load_vec(p + i * each, v);
    load_vec(p + i * each + HALF, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] += v[j], u[j] += w[j];
  }
  if (a.kept) Kept<T>(a.kept, s.rows, s.hidden).store(m * pad + n, g, u);
  activate<T>(a.act, g, act, slope);
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] = act[j] * u[j];
  store_upto((T*)a.h + m * s.hidden + n, left, g);
}

template <typename T, int SIDE>
static void wide_launch(int mode, const GatedWide& a, hipStream_t st) {
  const int join = a.cut * (SIDE * SIDE / 8 / 256);
  if (mode == kWideFwd) {
    k_wide<T, kWideFwd, SIDE><<<a.whole + a.cut * a.shares, kWideThreads, 0, st>>>(a);
    if (join) k_wide_join_fwd<T, SIDE><<<join / 2, 256, 0, st>>>(a);
  } else if (mode == kWideGrad) {
    k_wide<T, kWideGrad, SIDE><<<a.mt * a.nt, kWideThreads, 0, st>>>(a);
  } else if (mode == kWideDx) {
    k_wide<T, kWideDx, SIDE><<<a.whole + a.cut * a.shares, kWideThreads, 0, st>>>(a);
    if (join) k_wide_join<T, kWideDx, SIDE><<<join, 256, 0, st>>>(a);
  } else {
    k_wide<T, kWideDw, SIDE><<<a.whole + a.cut * a.shares, kWideThreads, 0, st>>>(a);
    if (join) k_wide_join<T, kWideDw, SIDE><<<join, 256, 0, st>>>(a);
  }
}

// How a product of mt x nt tiles is cut.  Work goes by CU: tiles that do not make up whole rounds of 256 are
// cut along K into the shares (each at least eight steps, or two of fp32's, which take four times as
// long) that end first by a model in steps of K: a CU takes its workgroups' steps, `open` for each
// one's first loads and last stores, a tenth more where one of 128 has the CU to itself (two fill each
// other's gaps; 256 always has), and for each share `part`, its sums' way through memory, beside the
// join's launch.  Fitted to fp32 (72 tiles of
// 188 steps: 3 shares 138 us, 7 118; 250 of 32: whole 72, 2 78; 128 of 128: 2 142, 4 137; 16 of
// 500: 16 73, 32 80; 141 of 94: whole 186, 3 135) and bf16 (256 tiles of 128, 88 steps: whole 51, 2
// 57).  A forward's cut tiles get their activation in the join: 100 x 4000 -> 1000 fp32 31 us against
// 225 in 64 x 64 tiles, bf16 17.5 against 27.8 uncut.
WideRounds gated_wide_rounds(int type, int side, int64_t mt, int64_t nt, int64_t steps) {
  const int64_t tiles = mt * nt, cut = tiles % 256;
  const double open = type == GSR_F32 ? 2. : side == 256 ? 3.5 : 4., part = type == GSR_F32 ? .015 : side == 256 ? .08 : .06;
  const double join = type == GSR_F32 ? 1.5 : side == 256 ? 2. : 6.;
  const int64_t least = type == GSR_F32 ? 2 : 8, most = steps / least < 64 ? steps / least : 64;
  int64_t shares = 1;
  double best = 0.;
  for (int64_t n = 1; cut && (n == 1 || n <= most); ++n) {
    const int64_t each = ceil_div64(cut * n, 256);   // workgroups a CU
    if (n > 1 && each > (side == 256 ? 1 : 2)) break;   // all run at once
    double cost = each * ((double)steps / n + open);
    if (each == 1 && side == 128 && tiles < 256) cost *= 1.1;
    if (n > 1) cost += join + part * cut * n;
    if (n == 1 || cost < best) best = cost, shares = n;
  }
  return shares > 1 ? WideRounds{(int)(tiles - cut), (int)cut, (int)shares} : WideRounds{(int)tiles, 0, 1};
}

// The same for dx and dW side by side (128), where all their workgroups run at once (else false).  Shares of one
// length in both, a little more than makes 512 of them, by the same model: of two workgroups a CU, the
// longer kind paired with the shorter where there are at most 256 of it.  Backward passes, side
// by side against one after the other: fp32 16000 x 256 -> 512 161 us against 173, 500 x 1000 -> 1000
// 53 against 62; bf16 777 x 509 -> 1363 23 against 32, 4096 x 256 -> 4096 89 against 96.
bool gated_wide_back_rounds(int type, const int64_t (&tiles)[2], const int64_t (&steps)[2], WideRounds (&r)[2]) {
  const bool f32 = type == GSR_F32;
  const double open = f32 ? 2. : 4., part = f32 ? .015 : .06, join = f32 ? 1.5 : 6.;
  const double all = (double)(tiles[0] * steps[0] + tiles[1] * steps[1]);
  const int64_t least = f32 ? 2 : 8;
  double best = 0.;
  for (int j = 0; j < 16; ++j) {
    const double length = all / 512 * (1. + j / 16.);
    int64_t n[2], count[2];
    double unit[2], cost = 0.;
    for (int i = 0; i < 2; ++i) {
      n[i] = (int64_t)(steps[i] / length) + 1;
      const int64_t most = steps[i] / least < 64 ? steps[i] / least : 64;
      n[i] = n[i] < most ? n[i] : most < 1 ? 1 : most;
      count[i] = tiles[i] * n[i];
      unit[i] = (double)steps[i] / n[i] + open;
      if (n[i] > 1) cost += part * count[i];
    }
    if (n[0] > 1 || n[1] > 1) cost += join;
    const int64_t total = count[0] + count[1];
    if (total > 512) continue;
    const int big = unit[1] > unit[0];
    cost += total <= 256 ? 1.1 * unit[big] : count[big] <= 256 ? unit[big] + unit[!big] : 2 * unit[big];
    if (best == 0. || cost < best) {
      best = cost;
      for (int k = 0; k < 2; ++k) r[k] = n[k] > 1 ? WideRounds{0, (int)tiles[k], (int)n[k]} : WideRounds{(int)tiles[k], 0, 1};
    }
  }
  return best > 0.;
}

static void wide_tiles(int mode, int side, const WideRounds& r, GatedWide* a) {
  const int64_t pad = gated_pad(a->s.hidden);
  a->mt = ceil_div(mode == kWideDw ? 2 * pad : a->s.rows, side);
  a->nt = mode <= kWideGrad ? ceil_div(pad, side / 2) : ceil_div(a->s.dim, side);
  a->whole = r.whole, a->cut = r.cut, a->shares = r.shares;
}

void gated_wide(int type, int mode, int side, GatedWide a, const WideRounds& r, hipStream_t st) {
  wide_tiles(mode, side, r, &a);
  if (mode == kWideGrad) a.whole = a.mt * a.nt, a.cut = 0;
  if (type == GSR_F32) {
    wide_launch<float, 128>(mode, a, st);
  } else if (type == GSR_BF16 && side == 256) {
    wide_launch<bf16, 256>(mode, a, st);
  } else if (type == GSR_BF16) {
    wide_launch<bf16, 128>(mode, a, st);
  } else if (side == 256) {
    wide_launch<f16, 256>(mode, a, st);
  } else {
    wide_launch<f16, 128>(mode, a, st);
  }
}

template <typename T>
static void wide_back_launch(const GatedWide& x, const GatedWide& w, hipStream_t st) {
  const int nx = x.whole + x.cut * x.shares, nw = w.whole + w.cut * w.shares, jx = x.cut * (128 * 128 / 8 / 256), jw = w.cut * (128 * 128 / 8 / 256);
  k_wide_back<T><<<nx + nw, kWideThreads, 0, st>>>(x, w, nx);
  if (jx + jw) k_wide_join_back<T><<<jx + jw, 256, 0, st>>>(x, w, jx);
}

void gated_wide_back(int type, GatedWide a, const WideRounds& rx, float* x_cuts, const WideRounds& rw, float* w_cuts, hipStream_t st) {
  GatedWide x = a, w = a;
  wide_tiles(kWideDx, 128, rx, &x);
  wide_tiles(kWideDw, 128, rw, &w);
  x.cuts = x_cuts, w.cuts = w_cuts;
  if (type == GSR_F32) {
    wide_back_launch<float>(x, w, st);
  } else if (type == GSR_BF16) {
    wide_back_launch<bf16>(x, w, st);
  } else {
    wide_back_launch<f16>(x, w, st);
  }
}

}  // namespace gsr
