// Launch of the gated block's products on square tiles of 256 or 128 (gated_wide.hip).
#pragma once

#include "gated.h"

namespace gsr {

enum { kWideFwd, kWideGrad, kWideDx, kWideDw };

// The tensors of one product, 16-bit, x, wg and wu 16-byte aligned with strides (in elements) that are
// multiples of 8, and kdim, the length of their rows, too: the block's dim, or it padded with zeros.
struct GatedWide {
  GatedShape s;
  int64_t kdim, x_stride, w_stride, dh_stride;
  const void *x, *wg, *wu, *bg, *bu, *dh;
  void *h, *dgu, *dx, *dwg, *dwu;
  float* parts;    // gradients: column sums [ceil(rows / side) * 2][2][hidden]; dx: [share][rows][dim]; dW:
                   // [share][2][hidden][dim]; or NULL
  int64_t share;   // dx: columns of dgu a share; dW: rows of x a share; multiples of 64
  int act, mt, nt;
};

void gated_wide(int type, int mode, int side, GatedWide a, int shares, hipStream_t st);

}  // namespace gsr
