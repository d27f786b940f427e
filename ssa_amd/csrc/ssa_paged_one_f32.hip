// The paged step's kernels of causal chunks and single tokens, f32 (a file of its own, so that the
// instantiations compile beside the others).

#include "ssa_paged_rows.h"

int ssa::paged_one_f32(tile::DenseParams& p, const PagedPlan& l, bool wide, bool zero_rows, char* ws, hipStream_t st) {
  return wide ? launch_rule<float, 128, kOne>(p, l, zero_rows, ws, st) : launch_rule<float, 64, kOne>(p, l, zero_rows, ws, st);
}
