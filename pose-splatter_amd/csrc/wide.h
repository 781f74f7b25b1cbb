// Products with fp32 sums in square tiles of 256 or 128: the parts of the gated block's main loop.
// Written for 16-bit matrices; fp32 ones (128 only) take 32 K a step in the place of 64 and
// 32x32x2 matrix instructions, four to each 16 bytes of an operand, and need no transposed reads.
//
// A workgroup of four waves owns a 256 x 256 tile, each wave a 128 x 128 quarter of 4 x 4 blocks
// of 32x32x16 matrix instructions: 256 accumulators a lane.  K advances 64 at a time; shared memory
// is a ring of five operand tiles (32 KB each, all of it): the two in use and three on their way,
// so a tile's loads have one to one and three quarters of a step to land.  A quarter that large reads
// 2 x 128 x 64 elements for 128 x 128 x 64 multiply-adds, 64 bytes of shared memory a cycle and
// CU at full matrix rate where 128 are available; eight waves of 128 x 64 would need 96 and leave
// none for the stores.  128 x 128 tiles (2 x 2 blocks a wave, two workgroups a CU) are for products
// of fewer tiles than CUs.
//
// Tiles come straight from global memory into shared memory (16 bytes a lane, no registers).  Each
// operand is read in the order it lies in memory:
//   K contiguous     rows of 64 K (128 bytes, a cache line); 16-byte chunk c of row r sits in slot
//                    c ^ (r % 8), so the 16-byte reads of eight neighbouring rows hit different banks
//   K across rows    rows of 256 (128) columns a K; chunk c of row k sits in slot
//                    c ^ (2 (k % 4) + 8 (k / 8 % 4 (% 2))); ds_read_b64_tr_b16 turns 4 K x 16 columns
//                    into the instruction's K-contiguous operand on the way out
// The pattern is made by choosing what each lane loads: shared memory itself is filled in lane
// order.  Loads past an operand's end return zeros (the buffer descriptor's bound), so no tile
// needs a special case; only K's own end inside a row is checked lane by lane.
#pragma once

#include "types.h"

namespace gsr {

template <typename T>
constexpr int kWideK = 128 / sizeof(T);   // K of a step: 128 bytes
constexpr int kWideSlots = 5, kWideThreads = 256;
constexpr uint32_t kWideNowhere = 0x80000000u;   // past every descriptor's end

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 wide_v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 wide_v8h __attribute__((ext_vector_type(8)));

// c += a b over 8 (fp32) or 16 K: 16 bytes of K a lane, the lower 32 lanes' first.
template <typename T>
__device__ __forceinline__ v16f wide_mma(v8s a, v8s b, v16f c) {
  if constexpr (__is_same(T, bf16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(wide_v8bf, a), __builtin_bit_cast(wide_v8bf, b), c, 0, 0, 0);
  } else if constexpr (__is_same(T, f16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(wide_v8h, a), __builtin_bit_cast(wide_v8h, b), c, 0, 0, 0);
  } else {
    const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[s], y[s], c, 0, 0, 0);
    return c;
  }
}

// Where a tile's loads come from: a buffer descriptor that starts at the tile's corner and holds
// `bytes` from there (loads past them return zeros), moved along by whole steps of K.
struct WideSource {
  uint32_t lo, hi, bytes;
  __device__ __forceinline__ WideSource(const void* corner, int64_t n)
      : lo((uint32_t)(uint64_t)corner), hi((uint32_t)((uint64_t)corner >> 32)), bytes((uint32_t)n) {}
  WideSource() = default;
  __device__ __forceinline__ void advance(uint32_t step) {
    const uint64_t b = ((uint64_t)hi << 32 | lo) + step;
    lo = (uint32_t)b;
    hi = (uint32_t)(b >> 32);
  }
  // of no length where `any` is false
  __device__ __forceinline__ v4i descriptor(bool any) const {
    return v4i{(int)lo, (int)hi, any ? (int)bytes : 0, 0x00027000};
  }
};

// 16 bytes a lane from src + off into shared memory at `lds` + `plus` (this wave's 1 KB, in lane
// order).  Written by hand because the compiler would wait for all loads before any read of
// shared memory; wide_wait() below is their wait.  They name no destination register.
__device__ __forceinline__ void wide_load(const v4i& src, uint32_t off, uint32_t lds, int plus) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(src),
               "n"(plus)
               : "memory", "scc");
}
// Until at most N of this wave's loads are in flight (they land in order), and its reads of shared
// memory are done.
template <int N>
__device__ __forceinline__ void wide_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Orders a wave's own reads and writes of shared memory (they complete in order; the compiler may
// not move them).
__device__ __forceinline__ void wide_fence() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// One operand's tile of SIDE rows (KC) or columns: this lane's places in it.
template <typename T, bool KC, int SIDE>
struct WideTile {
  static constexpr int BYTES = SIDE * 128, LOADS = BYTES / 4096, BLOCKS = SIDE / 64, ES = sizeof(T);
  static constexpr int ROW = SIDE * ES;   // bytes of a K row (K across rows)
  static constexpr int READS = KC ? 4 : ES == 4 ? BLOCKS : 2 * BLOCKS;
  uint32_t at[LOADS];   // byte offsets of the lane's loads from the tile's corner
  int k;                // KC: the loads' first K
  uint32_t read[READS];   // byte offsets of its reads: per quarter of a step (KC), or per (K parity and) block

  // origin: the wave's first row (KC) or column of the tile's
  __device__ __forceinline__ void init(int64_t stride_bytes, int origin) {
    const int t = threadIdx.x, l = t % 64;
    if constexpr (KC) {
      const int c = t % 8 ^ (t / 8 & 7);
      k = c * (16 / ES);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) at[j] = (uint32_t)((j * 32 + t / 8) * stride_bytes + c * 16);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) read[kk] = (origin + l % 32) * 128 + ((kk * 2 + l / 32) ^ (l & 7)) * 16;
    } else {
      constexpr int SLOTS = ROW / 16, EACH = 256 / SLOTS;   // 16-byte slots a K row, K rows a load
      constexpr int MASK = ES == 4 ? 0 : SIDE == 256 ? 3 : 1, MIX = ES == 4 ? 0 : 3;   // (fp32: chunks in order)
      k = 0;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int kr = j * EACH + t / SLOTS;
        at[j] = (uint32_t)(kr * stride_bytes + (t % SLOTS ^ (kr & MIX) * 2 ^ (kr >> 3 & MASK) * 8) * 16);
      }
      if constexpr (ES == 4) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) read[b] = l / 32 * 4 * ROW + (origin + b * 32 + l % 32) * 4;
      } else {
        const int g = l / 16, row = l % 16 / 4;   // K row of the lane's 4 x 16 piece
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            const int c = origin / 8 + b * 4 + g % 2 * 2 + l % 4 / 2;
            read[p * BLOCKS + b] = (g / 2 * 8 + row) * ROW + (c ^ row * 2 ^ (p * 2 + g / 2 & MASK) * 8) * 16 + l % 2 * 8;
          }
      }
    }
  }

  // The lane's j-th load's offset, where `left` K are left at the tile's start.
  __device__ __forceinline__ uint32_t offset(int j, int left) const { return !KC || k < left ? at[j] : kWideNowhere; }

  // The operand of the 32 rows from the wave's origin + `off` (a multiple of 32, below SIDE / 2 where
  // K runs across rows) and quarter kk of the step's K.
  __device__ __forceinline__ v8s operand(const char* lds, int off, int kk) const {
    if constexpr (KC) {
      return *(const v8s*)(lds + read[kk] + off * 128);
    } else if constexpr (ES == 4) {
      const char* p = lds + read[off / 32] + kk * 8 * ROW;
      return __builtin_bit_cast(v8s, v4f{*(const float*)p, *(const float*)(p + ROW), *(const float*)(p + 2 * ROW),
                                         *(const float*)(p + 3 * ROW)});
    } else {
      typedef __attribute__((address_space(3))) v4s lds_v4s;
      const char* p = lds + read[kk % 2 * BLOCKS + off / 32] + kk * 16 * ROW;
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p);
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 4 * ROW));
      return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Workgroup `id` of a launch -> its tile.  Workgroups go round the eight XCDs in turn: each XCD gets a
// run of neighbouring tiles, in groups of eight tile rows, so that its L2 holds what they share.
__device__ __forceinline__ void wide_tile_of(int id, int mt, int nt, int* m, int* n) {
  const int total = mt * nt, q = total / 8, r = total % 8, xcd = id % 8;
  const int pos = (xcd < r ? xcd * (q + 1) : r + xcd * q) + id / 8;
  const int group = pos / (8 * nt), first = group * 8, rows = mt - first < 8 ? mt - first : 8, in = pos - group * 8 * nt;
  *m = first + in % rows;
  *n = in / rows;
}

}  // namespace gsr
