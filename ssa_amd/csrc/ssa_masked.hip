// Dense softmax attention with a key interval per row, forward
// (ssa_masked_attention), and the intervals of the usual masks (ssa_mask_spans).
// The kernel is dense_rows_kernel (ssa_dense_rows.h).

#include "ssa_masked_rows.h"

namespace ssa {
namespace {

using namespace tile;

// One thread a row: the document that holds it (the last start at or before it,
// by bisection) and the keys it sees there.
__global__ __launch_bounds__(256) void mask_spans_kernel(const int32_t* starts, int docs, const int32_t* prefix,
                                                         int64_t batch, int64_t n, int64_t n_q, int64_t q_pos0,
                                                         int causal, int64_t window, int64_t sinks, int2* out) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= batch * n_q) return;
  const int64_t b = t / n_q, pos = q_pos0 + (t - b * n_q);
  int64_t lo = 0, end = n;
  int at = 0;
  if (starts != nullptr) {
    const int32_t* s = starts + b * (docs + 1);
    int x = 0, y = docs + 1;  // the first start past the row
    while (x < y) {
      const int mid = (x + y) >> 1;
      if (s[mid] <= pos)
        x = mid + 1;
      else
        y = mid;
    }
    at = x - 1;
    if (at < 0 || at >= docs) {
      if (window > 0) {
        reinterpret_cast<int4*>(out)[t] = make_int4(0, 0, 0, 0);
      } else {
        out[t] = make_int2(0, 0);
      }
      return;
    }
    lo = max(s[at], 0);
    end = min(static_cast<int64_t>(s[at + 1]), n);
  }
  int64_t hi = end;
  if (causal) {
    hi = pos + 1;
    if (prefix != nullptr) hi = max(hi, lo + prefix[b * docs + at]);
    hi = min(hi, end);
  }
  if (window > 0) {  // the window's keys, and the first ones (and the prefix) before it
    int64_t far = min(lo + sinks, pos + 1);
    if (prefix != nullptr) far = max(far, lo + prefix[b * docs + at]);
    int64_t from = max(lo, pos + 1 - window), to = min(pos + 1, end);
    far = min(far, end);
    if (far >= from) {  // (they meet)
      from = lo;
      to = max(to, far);
      far = lo;
    }
    int4 s = make_int4(0, 0, 0, 0);
    if (to > from) {
      s.x = static_cast<int>(from);
      s.y = static_cast<int>(to);
    }
    if (far > lo) {
      s.z = static_cast<int>(lo);
      s.w = static_cast<int>(far);
    }
    reinterpret_cast<int4*>(out)[t] = s;
    return;
  }
  out[t] = hi > lo ? make_int2(static_cast<int>(lo), static_cast<int>(hi)) : make_int2(0, 0);
}

}  // namespace
}  // namespace ssa

using namespace ssa;
using namespace ssa::tile;

static int mask_spans(const int32_t* doc_starts, int docs, const int32_t* prefix_lens, int64_t batch, int64_t n, int64_t n_q,
                      int64_t q_pos0, int causal, int64_t window, int64_t sinks, int32_t* spans, void* stream) {
  if (batch < 0 || n < 0 || n_q < 0 || q_pos0 < 0 || n >= (int64_t(1) << 31))
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans: bad shape batch=%lld n=%lld n_q=%lld q_pos0=%lld",
                (long long)batch, (long long)n, (long long)n_q, (long long)q_pos0);
  if (docs < 1) return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans: docs=%d must be positive", docs);
  if (doc_starts == nullptr && docs != 1)
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans: without doc_starts a sequence is one document");
  if (batch == 0 || n_q == 0) return SSA_OK;
  if (!spans) return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans: null pointer");
  const int64_t grid = ceil_div(batch * n_q, 256);
  if (grid > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "ssa_mask_spans: too many rows");
  mask_spans_kernel<<<dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream)>>>(
      doc_starts, docs, prefix_lens, batch, n, n_q, q_pos0, causal != 0, window, sinks, reinterpret_cast<int2*>(spans));
  return check_launch("ssa_mask_spans");
}

extern "C" int ssa_mask_spans(const int32_t* doc_starts, int docs, const int32_t* prefix_lens, int64_t batch,
                              int64_t n, int64_t n_q, int64_t q_pos0, int causal, int32_t* spans, void* stream) {
  return mask_spans(doc_starts, docs, prefix_lens, batch, n, n_q, q_pos0, causal, 0, 0, spans, stream);
}

extern "C" int ssa_mask_spans_window(const int32_t* doc_starts, int docs, const int32_t* prefix_lens, int64_t batch,
                                     int64_t n, int64_t n_q, int64_t q_pos0, int64_t window, int64_t sinks, int32_t* spans,
                                     void* stream) {
  const int64_t most = int64_t(1) << 31;  // (past every key)
  if (window < 1 || sinks < 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans_window: window must be positive and sinks not negative");
  if (reinterpret_cast<uintptr_t>(spans) % 16 != 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "ssa_mask_spans_window: spans must be aligned to 16 bytes");
  return mask_spans(doc_starts, docs, prefix_lens, batch, n, n_q, q_pos0, 1, window < most ? window : most,
                    sinks < most ? sinks : most, spans, stream);
}

namespace ssa {

int score_rule(const char* fn, float scale_div, float softcap, const float* slopes, tile::ScoreRule* r) {
  if (!(scale_div > 0.0f) || !isfinite(scale_div))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: scale_div must be positive and finite", fn);
  if (!(softcap >= 0.0f) || !isfinite(softcap))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: softcap must be finite and not negative (0: none)", fn);
  // (so that c1, c2 and a score times c1 are normal fp32 numbers)
  const double both = softcap > 0.0f ? static_cast<double>(scale_div) * softcap : scale_div;
  auto out = [](double x) { return x < 1e-30 || x > 1e30; };
  if (out(scale_div) || out(both) || (softcap > 0.0f && out(softcap)))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: scale_div, softcap and their product must lie in the range of 1e-30 to 1e30", fn);
  r->cap = softcap > tile::kMostDirectCap ? tile::kSeries : (softcap > 0.0f ? tile::kDirect : tile::kNoCap);
  r->c1 = r->cap ? static_cast<float>(1.0 / (static_cast<double>(scale_div) * softcap))
                 : static_cast<float>(1.4426950408889634074 / scale_div);
  r->c2 = static_cast<float>(1.4426950408889634074 * softcap);
  r->slopes = slopes;
  return SSA_OK;
}

int check_heads(const char* fn, int dtype, int h_q, int h_kv, int d) {
  if (dtype != SSA_DTYPE_F32 && dtype != SSA_DTYPE_BF16)
    return fail(SSA_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", fn);
  if (h_q <= 0 || h_kv <= 0 || d <= 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape h_q=%d h_kv=%d d=%d", fn, h_q, h_kv, d);
  if (h_q % h_kv != 0) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: h_q=%d must be divisible by h_kv=%d", fn, h_q, h_kv);
  if (h_q / h_kv > 16) return fail(SSA_ERR_UNSUPPORTED, "%s: GQA group size %d > 16", fn, h_q / h_kv);
  if (d % 8 != 0 || d > 128) return fail(SSA_ERR_UNSUPPORTED, "%s: head_dim %d must be a multiple of 8, at most 128", fn, d);
  return SSA_OK;
}

// Rows of 16 bytes: the base and every stride a multiple of 16 bytes.
int check_aligned(const char* fn, const char* name, int dtype, const void* ptr, int64_t s0, int64_t s1, int64_t s2) {
  const int64_t e = dtype == SSA_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0 || (s0 * e) % 16 != 0 || (s1 * e) % 16 != 0 || (s2 * e) % 16 != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s must have rows aligned to 16 bytes", fn, name);
  // (a tile's rows are addressed by 32-bit offsets, heads by 64-bit pointers)
  if (s1 < 0 || s2 < 0 || s1 > tile::kMostRowBytes / e)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s must have row strides of 0 to %lld bytes, and head strides from 0", fn, name,
                (long long)tile::kMostRowBytes);
  return SSA_OK;
}

}  // namespace ssa

extern "C" size_t ssa_masked_attention_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q, int h_q, int h_kv,
                                                       int d) {
  if (batch <= 0 || n <= 0 || n_q <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return 0;
  if (batch > 0x7FFFFFFF || n > 0x7FFFFF00 || n_q > 0x7FFFFF00) return 0;  // (what the call refuses)
  const int s = dense_split(n_q * (h_q / h_kv), batch * h_kv, n, n_q, dtype == SSA_DTYPE_F32, d > 64, false).parts;
  if (s <= 1) return 0;
  return static_cast<size_t>(s) * batch * n_q * h_q * ((d <= 64 ? 64 : 128) + 2) * sizeof(float);
}

static int forward(const char* fn, bool two, const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n,
                                    int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                                    int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn,
                                    int64_t v_sh, const int32_t* spans, float scale_div, float softcap,
                                    const float* slopes, void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh,
                                    void* out_low, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_heads(fn, dtype, h_q, h_kv, d)) return rc;
  if (batch < 0 || n < 0 || n_q < 0 || q_pos0 < 0 || batch > 0x7FFFFFFF)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape batch=%lld n=%lld n_q=%lld q_pos0=%lld", fn, (long long)batch,
                (long long)n, (long long)n_q, (long long)q_pos0);
  // keys, positions and packed rows are 32-bit in the kernel, with a tile to spare
  if (n > 0x7FFFFF00 || q_pos0 + n_q > 0x7FFFFF00 || n_q * (h_q / h_kv) > 0x7FFFFF00)
    return fail(SSA_ERR_UNSUPPORTED, "%s: sequences must be shorter than 2^31 / group size", fn);
  tile::DenseParams p{};
  if (int rc = score_rule(fn, scale_div, softcap, slopes, &p.rule)) return rc;
  if (batch == 0 || n_q == 0) return SSA_OK;
  if (!q || !out || (n > 0 && (!k || !v))) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, "q", dtype, q, q_sb, q_sn, q_sh)) return rc;
  if (int rc = check_aligned(fn, "k", dtype, k, k_sb, k_sn, k_sh)) return rc;
  if (int rc = check_aligned(fn, "v", dtype, v, v_sb, v_sn, v_sh)) return rc;
  if (int rc = check_aligned(fn, "out", dtype, out, o_sb, o_sn, o_sh)) return rc;
  if (int rc = check_aligned(fn, "out_low", dtype, out_low, 0, 0, 0)) return rc;
  if (two && (spans == nullptr || reinterpret_cast<uintptr_t>(spans) % 16 != 0))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: spans must be given, aligned to 16 bytes", fn);
  p.q = q; p.k = k; p.v = v; p.out = out; p.out_low = out_low; p.lse = lse;
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh;
  p.k_sb = k_sb; p.k_sn = k_sn; p.k_sh = k_sh;
  p.v_sb = v_sb; p.v_sn = v_sn; p.v_sh = v_sh;
  p.o_sb = o_sb; p.o_sn = o_sn; p.o_sh = o_sh;
  p.n = n; p.n_q = n_q; p.q_pos0 = q_pos0;
  p.batch = static_cast<int>(batch); p.h_q = h_q; p.h_kv = h_kv; p.g = h_q / h_kv; p.d = d;
  p.spans = reinterpret_cast<const int2*>(spans);
  const DenseSplit cut = dense_split(n_q * p.g, batch * h_kv, n, n_q, dtype == SSA_DTYPE_F32, d > 64, false);
  p.splits = cut.parts;
  if (p.splits > 1) {
    const size_t need = ssa_masked_attention_workspace_bytes(dtype, batch, n, n_q, h_q, h_kv, d);
    if (workspace == nullptr || workspace_bytes < need)
      return fail(SSA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", fn, need,
                  workspace == nullptr ? size_t(0) : workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(SSA_ERR_INVALID_ARGUMENT, "%s: workspace must be aligned to 16 bytes", fn);
    p.part_rows = batch * n_q * h_q;
    p.split_len = ceil_div(ceil_div(n, p.splits), 64) * 64;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * p.part_rows * (d <= 64 ? 64 : 128);
  }
  hipStream_t st = as_stream(stream);
  if (two) return dtype == SSA_DTYPE_F32 ? masked_two_f32(p, cut.kw, st) : masked_two_bf16(p, cut.kw, st);
  if (dtype == SSA_DTYPE_F32)
    return d <= 64 ? launch_rows_rule<float, 64, kOne>(p, cut.kw, st) : launch_rows_rule<float, 128, kOne>(p, cut.kw, st);
  return d <= 64 ? launch_rows_rule<uint16_t, 64, kOne>(p, cut.kw, st) : launch_rows_rule<uint16_t, 128, kOne>(p, cut.kw, st);
}

extern "C" int ssa_masked_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n,
                                    int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                                    int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn,
                                    int64_t v_sh, const int32_t* spans, float scale_div, float softcap,
                                    const float* slopes, void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh,
                                    void* out_low, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return forward("ssa_masked_attention", false, q, k, v, dtype, batch, n, n_q, q_pos0, h_q, h_kv, d, q_sb, q_sn, q_sh, k_sb, k_sn,
                 k_sh, v_sb, v_sn, v_sh, spans, scale_div, softcap, slopes, out, o_sb, o_sn, o_sh, out_low, lse, workspace,
                 workspace_bytes, stream);
}

extern "C" int ssa_masked_attention_two(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n,
                                    int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                                    int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn,
                                    int64_t v_sh, const int32_t* spans, float scale_div, float softcap,
                                    const float* slopes, void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh,
                                    void* out_low, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return forward("ssa_masked_attention_two", true, q, k, v, dtype, batch, n, n_q, q_pos0, h_q, h_kv, d, q_sb, q_sn, q_sh, k_sb, k_sn,
                 k_sh, v_sb, v_sn, v_sh, spans, scale_div, softcap, slopes, out, o_sb, o_sn, o_sh, out_low, lse, workspace,
                 workspace_bytes, stream);
}
