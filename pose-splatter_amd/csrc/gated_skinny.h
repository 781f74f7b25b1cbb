// Launch of the gated block's projections of few rows (gated_skinny.hip).
#pragma once

#include "gated.h"

namespace gsr {

constexpr int kSkinnyRows = 64;

struct GatedSkinny {
  GatedShape s;   // rows <= kSkinnyRows
  const void *x, *wg, *wu, *bg, *bu, *dh;
  int64_t x_stride, dh_stride;
  void *h, *dgu;   // one of them: the forward, or the gradients of the projections
  float* parts;    // gradients: column sums [2][hidden], or NULL
  int act;
  bool dgu32;      // dgu is written in fp32
  void* kept;      // forward: NULL, or what it keeps of the projections (Kept)
};

void gated_skinny(int type, const GatedSkinny& a, hipStream_t st);

}  // namespace gsr
