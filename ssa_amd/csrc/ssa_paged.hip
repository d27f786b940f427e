// Attention of new tokens over a paged K/V cache (ssa_paged_step): a ragged batch
// of sequences, each with its new tokens' rows appended to its pages and attended
// over everything it has cached, causally.
//
//   append       blocks that copy the new rows to their pages, 16
//                bytes a thread; the attention reads them from the call's k and v, so
//                that nothing waits for the copies
//   few rows     sequences with at most 32 rows (tokens x heads of a group) per KV
//                head, single tokens above all: few_rows
//   many rows    chunks: dense_rows (ssa_dense_rows.h) over pages
//   few codes    at most 16 bf16 rows of one or two new tokens over pages of 8 bits: few_codes
//
// all in one launch, and the parts that sequences were cut into joined in a second.  Where
// the caller says that out holds nothing, blocks of the second (of the first, of calls
// without) write zeros to the rows of out that nothing else writes.
//
// few_rows reads K and V once and is bound by that.  The rows fill one
// MFMA column block; the block's four waves take every fourth 32-key tile of its
// part of the sequence, each through LDS of its own (whole rows loaded, so that
// every load instruction reads contiguous lines; the next tile's loads are in
// flight while a tile is used, and its pages are looked up a tile earlier still),
// and join their running sums through LDS at the end.  32 sequences of up to 8192
// cached tokens, 32 / 8 heads, bf16: 139 us, 4.6 TB/s of K and V (a large copy: 4.95);
// one of 131072, 16 / 2 heads: 28 us, 4.8 TB/s, and 9 us for the join of its 256 parts.
// One short sequence waits for memory four times in a row (table, page, K and V, out):
// 203 tokens, 8 / 2 heads, fp32, 12.4 us.
//
// ssa_paged_step_general adds windows, drafted trees and pages of 8 bits to the same launch: rows
// that see two intervals of keys (and, of a tree, a word of drafts) walk the tiles of both.
//
// The kernels are in ssa_paged_rows.h; ssa_paged_one_*.hip, ssa_paged_two_*.hip and
// ssa_paged_held_*.hip compile them.

#include <math.h>

#include "ssa_cuts.h"
#include "ssa_dense_rows.h"
#include "ssa_internal.h"

using namespace ssa;

extern "C" size_t ssa_paged_step_workspace_bytes(int dtype, int64_t tokens, int64_t batch, int h_q, int h_kv, int d,
                                                 int64_t max_new, int64_t max_len) {
  if (tokens <= 0 || batch <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0 || max_new <= 0 || max_len <= 0) return 0;
  // (what the call refuses: products of these would overflow, to a division by zero at worst)
  if (tokens > 0x7FFFFF00 || batch > 0x7FFFFF || max_len > 0x7FFFFF00) return 0;
  return paged_plan(dtype, tokens, batch, h_q, h_kv, d, max_new, max_len).bytes;
}

extern "C" size_t ssa_paged_step_general_workspace_bytes(int dtype, int page_dtype, int64_t tokens, int64_t batch, int h_q,
                                                         int h_kv, int d, int64_t max_new, int64_t max_len, int64_t window,
                                                         int64_t sinks) {
  if (tokens <= 0 || batch <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0 || max_new <= 0 || max_len <= 0) return 0;
  if (tokens > 0x7FFFFF00 || batch > 0x7FFFFF || max_len > 0x7FFFFF00 || window < 0 || sinks < 0) return 0;  // (what the call refuses)
  max_new = max_new < tokens ? max_new : tokens;
  return paged_plan(dtype, tokens, batch, h_q, h_kv, d, max_new, seen_len(max_len, max_new, window, sinks), 128,
                    codes_call(dtype, page_dtype, max_new, h_q / h_kv, d)).bytes;
}

namespace {

// What ssa_paged_step_general has beyond ssa_paged_step.
struct General {
  int64_t window, sinks;
  const int32_t* parents;
  int page_dtype;
  const float *k_scales, *v_scales;
  int64_t ks_sp, ks_st, ks_sh, vs_sp, vs_st, vs_sh;
};

// Pools of 8 bits: rows aligned to 8 bytes, a scale a row.
int check_codes(const char* fn, const char* name, const void* ptr, int64_t s0, int64_t s1, int64_t s2, const float* scales,
                int64_t c0, int64_t c1, int64_t c2) {
  if (reinterpret_cast<uintptr_t>(ptr) % 8 != 0 || s0 % 8 != 0 || s1 % 8 != 0 || s2 % 8 != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s of 8 bits must have rows aligned to 8 bytes", fn, name);
  if (s0 < 0 || s1 < 0 || s2 < 0 || s1 > tile::kMostRowBytes)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s must have row strides of 0 to %lld bytes, and other strides from 0", fn, name,
                (long long)tile::kMostRowBytes);
  if (scales == nullptr || reinterpret_cast<uintptr_t>(scales) % 4 != 0 || c0 < 0 || c1 < 0 || c2 < 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: %s of 8 bits need fp32 scales, with strides from 0", fn, name);
  return SSA_OK;
}

}  // namespace

static int paged_step(const char* fn, bool zero_rows, const General& x, const void* q, const void* k, const void* v, int dtype,
                      int64_t tokens, int64_t batch, int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st,
                      int64_t k_sh, int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages,
                      int page_size, int64_t kp_sp, int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st,
                      int64_t vp_sh, const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                      const int32_t* cached, int64_t max_new, int64_t max_len, float scale_div, float softcap,
                      const float* slopes, void* out, int64_t o_st, int64_t o_sh, int32_t* error_flag, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (int rc = check_heads(fn, dtype, h_q, h_kv, d)) return rc;
  const bool held = x.page_dtype == SSA_DTYPE_I8 || x.page_dtype == SSA_DTYPE_E4M3;
  if (!held && x.page_dtype != dtype)
    return fail(SSA_ERR_UNSUPPORTED, "%s: pages hold q's type, int8 or e4m3", fn);
  if (x.window < 0 || x.sinks < 0 || (x.sinks > 0 && x.window == 0))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: window must be positive (0: none), and sinks go with a window", fn);
  if (tokens < 0 || batch < 0 || num_pages < 0 || max_pages < 0 || max_new < 0 || max_len < 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape tokens=%lld batch=%lld num_pages=%lld max_pages=%d", fn,
                (long long)tokens, (long long)batch, (long long)num_pages, max_pages);
  if (page_size < 8 || page_size > 4096 || (page_size & (page_size - 1)) != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: page_size %d must be a power of 2 in [8, 4096]", fn, page_size);
  if (tokens > 0x7FFFFF00 || tokens * (h_q / h_kv) > 0x7FFFFF00 || batch > 0x7FFFFF || num_pages > 0x7FFFFFFF || max_len > 0x7FFFFF00 ||
      static_cast<int64_t>(max_pages) * page_size > 0x7FFFFF00)
    return fail(SSA_ERR_UNSUPPORTED, "%s: sequences must be shorter than 2^31 / group size", fn);
  tile::DenseParams p{};
  if (int rc = score_rule(fn, scale_div, softcap, slopes, &p.rule)) return rc;
  if (tokens == 0 || batch == 0) return SSA_OK;
  if (max_new < 1 || max_len < 1 || num_pages < 1 || max_pages < 1)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: max_new, max_len, num_pages and max_pages must be positive", fn);
  if (!q || !k_pages || !v_pages || !table || !starts || !cached || !out || (k == nullptr) != (v == nullptr))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, "q", dtype, q, 0, q_st, q_sh)) return rc;
  if (int rc = check_aligned(fn, "k", dtype, k, 0, k_st, k_sh)) return rc;
  if (int rc = check_aligned(fn, "v", dtype, v, 0, v_st, v_sh)) return rc;
  if (held) {
    if (int rc = check_codes(fn, "k_pages", k_pages, kp_sp, kp_st, kp_sh, x.k_scales, x.ks_sp, x.ks_st, x.ks_sh)) return rc;
    if (int rc = check_codes(fn, "v_pages", v_pages, vp_sp, vp_st, vp_sh, x.v_scales, x.vs_sp, x.vs_st, x.vs_sh)) return rc;
  } else {
    if (int rc = check_aligned(fn, "k_pages", dtype, k_pages, kp_sp, kp_st, kp_sh)) return rc;
    if (int rc = check_aligned(fn, "v_pages", dtype, v_pages, vp_sp, vp_st, vp_sh)) return rc;
  }
  if (int rc = check_aligned(fn, "out", dtype, out, 0, o_st, o_sh)) return rc;
  max_new = max_new < tokens ? max_new : tokens;
  if (x.parents != nullptr && max_new > tile::kDrafts)
    return fail(SSA_ERR_UNSUPPORTED, "%s: a tree has at most %d new tokens a sequence, max_new is %lld", fn, tile::kDrafts,
                (long long)max_new);
  // (a window that no sequence reaches is none)
  const int64_t window = x.window < max_len ? x.window : 0;
  const bool two = held || window > 0 || x.parents != nullptr;
  const PagedPlan l = paged_plan(dtype, tokens, batch, h_q, h_kv, d, max_new, seen_len(max_len, max_new, x.window, x.sinks),
                                 two ? 128 : 64, codes_call(dtype, x.page_dtype, max_new, h_q / h_kv, d));
  if (l.bytes > 0 && (workspace == nullptr || workspace_bytes < l.bytes))
    return fail(SSA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", fn, l.bytes,
                workspace == nullptr ? size_t(0) : workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: workspace must be aligned to 16 bytes", fn);
  p.q = q; p.k = k_pages; p.v = v_pages; p.out = out;
  p.q_sn = q_st; p.q_sh = q_sh;
  p.k_sb = kp_sp; p.k_sn = kp_st; p.k_sh = kp_sh;
  p.v_sb = vp_sp; p.v_sn = vp_st; p.v_sh = vp_sh;
  p.o_sn = o_st; p.o_sh = o_sh;
  p.n_q = tokens;
  p.batch = static_cast<int>(batch); p.h_q = h_q; p.h_kv = h_kv; p.g = h_q / h_kv; p.d = d;
  p.table = table; p.starts = starts; p.cached = cached; p.table_stride = table_stride;
  p.max_pages = max_pages; p.num_pages = static_cast<int>(num_pages);
  while ((1 << p.page_log2) < page_size) ++p.page_log2;
  p.few_rows = kFew;
  p.max_new = max_new; p.max_len = max_len;
  p.error_flag = error_flag;
  p.k_new = k; p.v_new = v;
  p.kn_st = k_st; p.kn_sh = k_sh; p.vn_st = v_st; p.vn_sh = v_sh;
  p.window = static_cast<int>(window);
  p.sinks = p.window > 0 ? static_cast<int>(x.sinks < 0x7FFFFFFF ? x.sinks : 0x7FFFFFFF) : 0;
  p.parents = x.parents;
  p.k_scale = x.k_scales; p.v_scale = x.v_scales;
  p.ks_sb = x.ks_sp; p.ks_sn = x.ks_st; p.ks_sh = x.ks_sh;
  p.vs_sb = x.vs_sp; p.vs_sn = x.vs_st; p.vs_sh = x.vs_sh;
  p.e4m3 = x.page_dtype == SSA_DTYPE_E4M3;
  hipStream_t st = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  const bool f32 = dtype == SSA_DTYPE_F32, wide = d > 64;
  if (held) return f32 ? paged_held_f32(p, l, wide, zero_rows, ws, st) : paged_held_bf16(p, l, wide, zero_rows, ws, st);
  if (two)
    return f32 ? paged_two_f32(p, l, wide, zero_rows, ws, st) : paged_two_bf16(p, l, wide, zero_rows, ws, st);
  return f32 ? paged_one_f32(p, l, wide, zero_rows, ws, st) : paged_one_bf16(p, l, wide, zero_rows, ws, st);
}

extern "C" int ssa_paged_step(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch,
                              int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                              int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages, int page_size,
                              int64_t kp_sp, int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh,
                              const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                              const int32_t* cached, int64_t max_new, int64_t max_len, float scale_div, float softcap,
                              const float* slopes, void* out, int64_t o_st, int64_t o_sh, int32_t* error_flag,
                              void* workspace, size_t workspace_bytes, void* stream) {
  General x{};
  x.page_dtype = dtype;
  return paged_step("ssa_paged_step", false, x, q, k, v, dtype, tokens, batch, h_q, h_kv, d, q_st, q_sh, k_st, k_sh, v_st,
                    v_sh, k_pages, v_pages, num_pages, page_size, kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh, table,
                    table_stride, max_pages, starts, cached, max_new, max_len, scale_div, softcap, slopes, out, o_st, o_sh,
                    error_flag, workspace, workspace_bytes, stream);
}

extern "C" int ssa_paged_step_zeroed(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch,
                                     int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                                     int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages,
                                     int page_size, int64_t kp_sp, int64_t kp_st, int64_t kp_sh, int64_t vp_sp,
                                     int64_t vp_st, int64_t vp_sh, const int32_t* table, int64_t table_stride,
                                     int max_pages, const int32_t* starts, const int32_t* cached, int64_t max_new,
                                     int64_t max_len, float scale_div, float softcap, const float* slopes, void* out,
                                     int64_t o_st, int64_t o_sh, int32_t* error_flag, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (tokens > 0 && batch == 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_paged_step_zeroed: rows without a sequence");
  General x{};
  x.page_dtype = dtype;
  return paged_step("ssa_paged_step_zeroed", true, x, q, k, v, dtype, tokens, batch, h_q, h_kv, d, q_st, q_sh, k_st, k_sh,
                    v_st, v_sh, k_pages, v_pages, num_pages, page_size, kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh, table,
                    table_stride, max_pages, starts, cached, max_new, max_len, scale_div, softcap, slopes, out, o_st, o_sh,
                    error_flag, workspace, workspace_bytes, stream);
}

extern "C" int ssa_paged_step_general(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch,
                                      int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                                      int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int page_dtype,
                                      float* k_scales, float* v_scales, int64_t num_pages, int page_size, int64_t kp_sp,
                                      int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh,
                                      int64_t ks_sp, int64_t ks_st, int64_t ks_sh, int64_t vs_sp, int64_t vs_st,
                                      int64_t vs_sh, const int32_t* table, int64_t table_stride, int max_pages,
                                      const int32_t* starts, const int32_t* cached, const int32_t* parents,
                                      int64_t max_new, int64_t max_len, int64_t window, int64_t sinks, float scale_div,
                                      float softcap, const float* slopes, void* out, int64_t o_st, int64_t o_sh,
                                      int zero_rows, int32_t* error_flag, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const General x{window, sinks, parents, page_dtype, k_scales, v_scales, ks_sp, ks_st, ks_sh, vs_sp, vs_st, vs_sh};
  if (zero_rows != 0 && tokens > 0 && batch == 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_paged_step_general: rows without a sequence");
  return paged_step("ssa_paged_step_general", zero_rows != 0, x, q, k, v, dtype, tokens, batch, h_q, h_kv, d, q_st, q_sh, k_st,
                    k_sh, v_st, v_sh, k_pages, v_pages, num_pages, page_size, kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh, table,
                    table_stride, max_pages, starts, cached, max_new, max_len, scale_div, softcap, slopes, out, o_st, o_sh,
                    error_flag, workspace, workspace_bytes, stream);
}
