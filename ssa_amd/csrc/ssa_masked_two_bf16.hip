// Dense attention whose rows see two key intervals, forward and backward, bf16 (a file of its
// own, so that the instantiations compile beside the others).

#include "ssa_masked_bwd_rows.h"
#include "ssa_masked_rows.h"

namespace ssa {

int masked_two_bf16(tile::DenseParams& p, int kw, hipStream_t st) {
  return p.d <= 64 ? launch_rows_rule<uint16_t, 64, kTwo>(p, kw, st) : launch_rows_rule<uint16_t, 128, kTwo>(p, kw, st);
}

int masked_two_backward_bf16(void* params, const BwdCut& cut, const TwoCut& two, hipStream_t st) {
  BwdParams& p = *static_cast<BwdParams*>(params);
  return p.d <= 64 ? launch_rule<uint16_t, 64, kTwo>(p, cut, two, st) : launch_rule<uint16_t, 128, kTwo>(p, cut, two, st);
}

}  // namespace ssa
