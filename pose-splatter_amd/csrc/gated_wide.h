// Launch of the gated block's products on square tiles of 256 or 128 (gated_wide.hip).
#pragma once

#include "gated.h"

namespace gsr {

enum { kWideFwd, kWideGrad, kWideDx, kWideDw };

// The tensors of one product: x, wg and wu 16-byte aligned, with strides (in elements) and kdim, the length
// of their rows, whole 16-byte pieces: the block's dim, or it padded with zeros.
struct GatedWide {
  GatedShape s;
  int64_t kdim, x_stride, w_stride, dh_stride;
  const void *x, *wg, *wu, *bg, *bu, *dh;
  void *h, *kept, *dgu, *dx, *dwg, *dwu;   // kept: NULL, or the forward's projections (Kept)
  float* parts;   // gradients: column sums [ceil(rows / side) * 2][2][hidden], or NULL
  float* cuts;    // forward, dx, dW: the cut tiles' sums [shares][cut][side][side]
  int act;
  bool dgu32;     // gradients: dgu is written in fp32
  int mt, nt, whole, cut, shares;   // set by the launch: tiles, and how they are cut (gated_wide_rounds)
};

// Tiles `whole` of a product are computed by one workgroup each, `cut` more by `shares` each.
struct WideRounds {
  int whole, cut, shares;
  int64_t bytes(int side) const { return cut ? (int64_t)cut * shares * side * side * 4 : 0; }
};
WideRounds gated_wide_rounds(int type, int side, int64_t mt, int64_t nt, int64_t steps);
bool gated_wide_back_rounds(int type, const int64_t (&tiles)[2], const int64_t (&steps)[2], WideRounds (&r)[2]);

// Steps of 128 bytes of K.
inline int64_t gated_wide_steps(int type, int64_t k) { return ceil_div64(k * (int64_t)type_size(type), 128); }

// side 128, or 256 in 16 bits
void gated_wide(int type, int mode, int side, GatedWide a, const WideRounds& r, hipStream_t st);

// dx and the weight gradients in one launch (side 128).
void gated_wide_back(int type, GatedWide a, const WideRounds& rx, float* x_cuts, const WideRounds& rw, float* w_cuts, hipStream_t st);

}  // namespace gsr
