// Gradients of dense attention with key intervals per row (ssa_masked_attention_backward,
// ssa_masked_attention_two_backward): the entry points and the kernels of one interval.  The
// kernels are in ssa_masked_bwd_rows.h.

#include "ssa_masked_bwd_rows.h"

namespace ssa {
namespace {

// dkv_kernel's offsets of a tile's 128 packed rows, ceil(127 / g) tokens and g - 1 heads from
// the first one's, have to stay within its resource.
int check_group(const char* fn, const char* name, int dtype, int g, int d, int64_t sn, int64_t sh) {
  const int64_t e = dtype == SSA_DTYPE_F32 ? 4 : 2, room = kAllBytes / e - d - (126 + g) / g * sn;
  if (g > 1 && sh > room / (g - 1))
    return fail(SSA_ERR_UNSUPPORTED, "%s: the heads of a group of %s must lie within 2 GiB", fn, name);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;


extern "C" size_t ssa_masked_attention_backward_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q,
                                                                int h_q, int h_kv, int d) {
  if (batch <= 0 || n <= 0 || n_q <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return 0;
  if (batch > 0x7FFFFFFF || n > 0x7FFFFF00 || n_q > 0x7FFFFF00) return 0;  // (what the call refuses)
  return bwd_cut(dtype, batch, n, n_q, h_q, h_kv, d).bytes;
}

extern "C" size_t ssa_masked_attention_two_backward_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q,
                                                                    int h_q, int h_kv, int d) {
  if (batch <= 0 || n <= 0 || n_q <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return 0;
  if (batch > 0x7FFFFFFF || n > 0x7FFFFF00 || n_q > 0x7FFFFF00) return 0;
  const BwdCut l = bwd_cut(dtype, batch, n, n_q, h_q, h_kv, d);
  return two_cut(l, dtype, batch, n, h_kv, d).bytes;
}

static int backward(
    const char* fn, bool two,
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q, int64_t q_pos0, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
    int64_t v_sn, int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes, const void* out,
    const void* out_low, int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_heads(fn, dtype, h_q, h_kv, d)) return rc;
  if (batch < 0 || n < 0 || n_q < 0 || q_pos0 < 0 || batch > 0x7FFFFFFF)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape batch=%lld n=%lld n_q=%lld q_pos0=%lld", fn, (long long)batch,
                (long long)n, (long long)n_q, (long long)q_pos0);
  if (n > 0x7FFFFF00 || q_pos0 + n_q > 0x7FFFFF00 || n_q * (h_q / h_kv) > 0x7FFFFF00)
    return fail(SSA_ERR_UNSUPPORTED, "%s: sequences must be shorter than 2^31 / group size", fn);
  BwdParams p{};
  if (int rc = score_rule(fn, scale_div, softcap, slopes, &p.rule)) return rc;
  if (batch == 0 || n == 0 || n_q == 0) {
    if (batch > 0 && (n > 0 || n_q > 0))
      return fail(SSA_ERR_INVALID_ARGUMENT, "%s: keys without rows, or rows without keys, have no gradient", fn);
    return SSA_OK;
  }
  if (!q || !k || !v || !out || !dout || !lse || !dq || !dk || !dv)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, "q", dtype, q, q_sb, q_sn, q_sh)) return rc;
  if (int rc = check_aligned(fn, "k", dtype, k, k_sb, k_sn, k_sh)) return rc;
  if (int rc = check_aligned(fn, "v", dtype, v, v_sb, v_sn, v_sh)) return rc;
  if (int rc = check_aligned(fn, "out", dtype, out, o_sb, o_sn, o_sh)) return rc;
  if (int rc = check_aligned(fn, "out_low", dtype, out_low, 0, 0, 0)) return rc;
  if (int rc = check_aligned(fn, "dout", dtype, dout, do_sb, do_sn, do_sh)) return rc;
  if (int rc = check_aligned(fn, "dq", dtype, dq, 0, 0, 0)) return rc;
  if (int rc = check_aligned(fn, "dk", dtype, dk, 0, 0, 0)) return rc;
  if (int rc = check_aligned(fn, "dv", dtype, dv, 0, 0, 0)) return rc;
  if (int rc = check_group(fn, "q", dtype, h_q / h_kv, d, q_sn, q_sh)) return rc;
  if (int rc = check_group(fn, "dout", dtype, h_q / h_kv, d, do_sn, do_sh)) return rc;
  if (two && (spans == nullptr || reinterpret_cast<uintptr_t>(spans) % 16 != 0))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: spans must be given, aligned to 16 bytes", fn);
  const BwdCut l = bwd_cut(dtype, batch, n, n_q, h_q, h_kv, d);
  const TwoCut two_l = two_cut(l, dtype, batch, n, h_kv, d);
  const size_t need = two ? two_l.bytes : l.bytes;
  if (two && two_l.key_blocks > 0x3FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many keys", fn);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", fn, need,
                workspace == nullptr ? size_t(0) : workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: workspace must be aligned to 16 bytes", fn);
  p.q = q; p.k = k; p.v = v; p.out = out; p.out_low = out_low; p.dout = dout; p.lse = lse;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh;
  p.k_sb = k_sb; p.k_sn = k_sn; p.k_sh = k_sh;
  p.v_sb = v_sb; p.v_sn = v_sn; p.v_sh = v_sh;
  p.o_sb = o_sb; p.o_sn = o_sn; p.o_sh = o_sh;
  p.do_sb = do_sb; p.do_sn = do_sn; p.do_sh = do_sh;
  p.n = n; p.n_q = n_q; p.q_pos0 = q_pos0;
  p.batch = static_cast<int>(batch); p.h_q = h_q; p.h_kv = h_kv; p.g = h_q / h_kv; p.d = d;
  p.spans = reinterpret_cast<const int2*>(spans);
  p.inv_scale = 1.0f / scale_div;
  char* ws = static_cast<char*>(workspace);
  p.stats = reinterpret_cast<float4*>(ws + l.stats);
  p.bounds = reinterpret_cast<int4*>(ws + l.bounds);
  p.groups = l.groups;
  p.splits = l.splits;
  hipStream_t st = as_stream(stream);
  if (two) {
    if (two_l.planned) {
      p.key_blocks = static_cast<int>(two_l.key_blocks);
      p.key_tiles = static_cast<int>(two_l.key_blocks / batch);
      p.extra = two_l.extra;
      p.counts = reinterpret_cast<int*>(ws + two_l.counts);
      p.entries = reinterpret_cast<int4*>(ws + two_l.entries);
      p.cut = reinterpret_cast<int4*>(ws + two_l.cut);
    }
    p.part_k = reinterpret_cast<float*>(ws + two_l.part);
    p.part_v = p.part_k + two_l.part_floats;
    return dtype == SSA_DTYPE_F32 ? masked_two_backward_f32(&p, l, two_l, st) : masked_two_backward_bf16(&p, l, two_l, st);
  }
  if (l.splits > 1) {
    p.part_k = reinterpret_cast<float*>(ws + l.part);
    p.part_v = p.part_k + static_cast<int64_t>(l.splits) * batch * n * h_kv * (d <= 64 ? 64 : 128);
  }
  if (dtype == SSA_DTYPE_F32) return d <= 64 ? launch_rule<float, 64, kOne>(p, l, two_l, st) : launch_rule<float, 128, kOne>(p, l, two_l, st);
  return d <= 64 ? launch_rule<uint16_t, 64, kOne>(p, l, two_l, st) : launch_rule<uint16_t, 128, kOne>(p, l, two_l, st);
}

extern "C" int ssa_masked_attention_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q, int64_t q_pos0, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
    int64_t v_sn, int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes, const void* out,
    const void* out_low, int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  return backward("ssa_masked_attention_backward", false, q, k, v, dtype, batch, n, n_q, q_pos0, h_q, h_kv, d, q_sb, q_sn, q_sh,
                  k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, spans, scale_div, softcap, slopes, out, out_low, o_sb, o_sn, o_sh, dout,
                  do_sb, do_sn, do_sh, lse, dq, dk, dv, workspace, workspace_bytes, stream);
}

extern "C" int ssa_masked_attention_two_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q, int64_t q_pos0, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
    int64_t v_sn, int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes, const void* out,
    const void* out_low, int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  return backward("ssa_masked_attention_two_backward", true, q, k, v, dtype, batch, n, n_q, q_pos0, h_q, h_kv, d, q_sb, q_sn, q_sh,
                  k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, spans, scale_div, softcap, slopes, out, out_low, o_sb, o_sn, o_sh, dout,
                  do_sb, do_sn, do_sh, lse, dq, dk, dv, workspace, workspace_bytes, stream);
}
