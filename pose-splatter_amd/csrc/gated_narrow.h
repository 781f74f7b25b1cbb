// Launch of the gated block's backward pass for narrow inputs (gated_narrow.hip).
#pragma once

#include "gated.h"

namespace gsr {

constexpr int64_t kNarrowDim = 15;   // the widest input they take

struct GatedNarrow {
  GatedShape s;   // dim <= kNarrowDim
  const void *x, *wg, *wu, *bg, *bu, *dh;
  int64_t x_stride, dh_stride;
  int act;
  void *dx, *dwg, *dwu, *dbg, *dbu;   // each may be NULL
  float *dw_parts, *dx_parts;         // of the sizes below
  int64_t cols;                       // set by the launch: columns of a workgroup, whole 16s
};

// Workgroups along the rows and the columns, and the floats of the partial sums: of the weights and
// biases [groups][2][hidden][dim and a bias, in fours], of dx [shares][rows][dim].
struct NarrowPlan {
  int64_t groups, shares;
  __host__ __device__ static int64_t width(int64_t dim) { return (dim + 4) / 4 * 4; }
  int64_t dw_floats(GatedShape s) const { return groups > 1 ? groups * 2 * s.hidden * width(s.dim) : 0; }
  int64_t dx_floats(GatedShape s) const { return shares > 1 ? shares * s.rows * s.dim : 0; }
};
NarrowPlan gated_narrow_plan(GatedShape s);

void gated_narrow(int type, GatedNarrow a, hipStream_t st);

}  // namespace gsr
