// The paged step's kernels of causal chunks and single tokens, bf16 (a file of its own, so that the
// instantiations compile beside the others).

#include "ssa_paged_rows.h"

int ssa::paged_one_bf16(tile::DenseParams& p, const PagedPlan& l, bool wide, bool zero_rows, char* ws, hipStream_t st) {
  return wide ? launch_rule<uint16_t, 128, kOne>(p, l, zero_rows, ws, st) : launch_rule<uint16_t, 64, kOne>(p, l, zero_rows, ws, st);
}
