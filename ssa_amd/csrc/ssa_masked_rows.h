// The forward kernel of ssa_masked_attention and ssa_masked_attention_two and how a call's cut and
// score rule choose it.
#pragma once

#include <math.h>

#include "ssa_cuts.h"
#include "ssa_dense_rows.h"
#include "ssa_internal.h"

namespace ssa {
namespace {

using namespace tile;

template <typename T, int D, int RULE, int KW, int VIEW>
__global__ __launch_bounds__(kThreads, (rows_per_cu<T, D, KW>())) void dense_rows_kernel(DenseParams p) {
  extern __shared__ __align__(16) char lds[];
  dense_rows<T, D, false, RULE, KW, false, VIEW>(p, blockIdx.x, lds);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void dense_join_kernel(DenseParams p) {
  dense_join<T, D>(p, static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6));
}

template <typename T, int D, int RULE, int KW, int VIEW>
int launch_rows(DenseParams& p, hipStream_t st) {
  const size_t bytes = rows_lds<T, D, KW>();
  if (int rc = reserve_lds(reinterpret_cast<const void*>(dense_rows_kernel<T, D, RULE, KW, VIEW>), bytes + 2048,
                           "ssa_masked_attention"))
    return rc;
  const int64_t blocks = ceil_div(p.n_q * p.g, rows_of(KW)) * p.batch * p.h_kv * p.splits;
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "ssa_masked_attention: too many rows");
  dense_rows_kernel<T, D, RULE, KW, VIEW><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), bytes, st>>>(p);
  if (int rc = check_launch("ssa_masked_attention")) return rc;
  if (p.splits > 1) {
    dense_join_kernel<T, D><<<dim3(static_cast<unsigned>(ceil_div(p.part_rows, kThreads / 64))), dim3(kThreads), 0, st>>>(p);
    return check_launch("ssa_masked_attention join");
  }
  return SSA_OK;
}

template <typename T, int D, int RULE, int VIEW>
int launch_rows_kw(DenseParams& p, int kw, hipStream_t st) {
  if constexpr (most_kw<T, D>() >= 4)
    if (kw == 4) return launch_rows<T, D, RULE, 4, VIEW>(p, st);
  return kw == 2 ? launch_rows<T, D, RULE, 2, VIEW>(p, st) : launch_rows<T, D, RULE, 1, VIEW>(p, st);
}

template <typename T, int D, int VIEW>
int launch_rows_rule(DenseParams& p, int kw, hipStream_t st) {
  switch (rule_kind<T>(p.rule)) {
    case kPlain: return launch_rows_kw<T, D, kPlain, VIEW>(p, kw, st);
    case kCap: return launch_rows_kw<T, D, kCap, VIEW>(p, kw, st);
    case kBias: return launch_rows_kw<T, D, kBias, VIEW>(p, kw, st);
    case kFar:
      if constexpr (sizeof(T) == 2) return launch_rows_kw<T, D, kFar, VIEW>(p, kw, st);
  }
  return fail(SSA_ERR_UNSUPPORTED, "no kernel for this rule of scores");
}

}  // namespace
}  // namespace ssa
