// The paged step's kernels of pages of 8-bit codes, f32 (a file of its own, so that the
// instantiations compile beside the others).

#include "ssa_paged_rows.h"

int ssa::paged_held_f32(tile::DenseParams& p, const PagedPlan& l, bool wide, bool zero_rows, char* ws, hipStream_t st) {
  return wide ? launch_rule<float, 128, kTwo, uint8_t>(p, l, zero_rows, ws, st) : launch_rule<float, 64, kTwo, uint8_t>(p, l, zero_rows, ws, st);
}
