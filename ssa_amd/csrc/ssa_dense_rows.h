// Softmax attention of many query rows over contiguous or paged keys: the
// forward kernel of ssa_masked_attention and of ssa_paged_step's chunks.
//
//   o_i = sum_j p_ij v_j,  p = softmax over lo_i <= j < hi_i of the score rule
//
// A block of four waves takes 128 rows of one KV head: a row is a (token, query
// head of the group) pair, tokens first, so that the g heads that share a key
// read its tile once and a causal block's diagonal is 128 / g tokens wide.  Where
// that leaves CUs idle, KW = 2 or 4 waves share 32 rows and take turns at the keys
// (64 or 32 rows a block; their sums meet in LDS).  Each wave keeps 32 rows: Q as B
// operands in registers, S^T = K Q^T with one row's scores down a lane's registers
// (the running maximum and sum need one exchange with the other half-wave), P^T as
// the B operand of O^T += V^T P^T without leaving its registers (ssa_tile.h).  K and V
// tiles of 64 keys (32 in fp32) pass through a double LDS buffer, the next tile's
// global loads in flight meanwhile.  Tiles that no row of a wave sees are skipped,
// tiles that every row sees whole take no mask arithmetic.
//
// Two waves a SIMD (250 registers each at d = 128) overlap one's products with the
// other's softmax, and the long calls run near the matrix cores' rate under the
// card's power limit (32 / 8 heads, bf16; an 8192^3 library product: 1.13 PFLOP/s):
//   16384 causal rows, d = 128        2.14 to 2.39 ms from card to card, 1.03 to 0.92 PFLOP/s
//   8192 x 8192, d = 128              1.12 ms, 0.98; d = 64 0.64 ms, 0.86 (the softmax is
//                                     the same work beside half the products)
//   2048 rows over 32768 paged keys   1.18 to 1.28 ms, 0.91 to 0.83
//   4096 x 4096, 16 / 4 heads, fp32   0.56 ms (d = 64), 123 of the product's 154 TFLOP/s
// Short ones are bound by each block's start (spans, Q, the first tile: 2 to 3 us) and
// by blocks of unlike lengths: twelve documents of 8192 tokens 155 us, 0.52 PFLOP/s.
//
// The running reference m is only moved when a tile's maximum exceeds it by more
// than 8 (in log2): weights then reach 2^8, which costs fp32 sums and bf16
// weights no relative precision, and most tiles rescale nothing.
//
// Of bf16 calls a weight (over 8-bit pages times its value's scale) is rounded to bf16 for its
// product with V, half a step of 2^-8 of it, as few_rows and few_codes do; scores, sums of weights and the
// products' sums are fp32.  An output is within 0.0024 of its scale of 64 bits so, its own rounding
// alone is 0.0017; products of fp32 weights run at an eighth of the rate.
//
// A masked key's weight is 0, but 0 times an infinity or NaN in its value row is
// not: a row whose accumulators end up other than finite is computed again key
// by key (exact_row), reading visible keys only.
//
// kTwo rows see more than one interval: two given ones, or over pages a sliding window
// and the first keys, and of drafted tokens in a tree their ancestors.  The block then
// walks the tiles of the two ranges that its rows see between them and no others, parts
// of the keys are equal shares of those tiles, and only tiles that some row does not see
// whole take the mask.  Pages of 8 bits (HELD) are widened to the products' type between
// the load and the LDS, where they are exact; a key's scale multiplies its score, a
// value's its weight, both in fp32.
#pragma once

#include <type_traits>

#include "ssa_cuts.h"
#include "ssa_tile.h"

namespace ssa {
namespace tile {

struct DenseParams {
  const void *q, *k, *v;
  void* out;
  void* out_low;  // nullable: what rounding out to bf16 leaves, in bf16 (out's strides)
  float* lse;  // nullable: [batch][h_q][n_q], log2 of the sum of weights (+inf: no key)
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, o_sb, o_sn, o_sh;
  int64_t n, n_q, q_pos0;  // keys; query tokens; position of query token 0
  int batch, h_q, h_kv, g, d;
  const int2* spans;  // null: causal by position (kTwo: pairs of them)
  ScoreRule rule;
  // kTwo over pages: keys back from a row that it sees (0: all) and first keys that all rows
  // see; parents of drafted tokens (nullable)
  int window, sinks;
  const int32_t* parents;
  // scales of pages of 8 bits, strides as the pools'
  const float *k_scale, *v_scale;
  int64_t ks_sb, ks_sn, ks_sh, vs_sb, vs_sn, vs_sh;
  int e4m3;
  // paged: k and v are the pools [pages][page rows][h_kv][d] (sb = page stride)
  const int32_t *table, *starts, *cached;
  int64_t table_stride;
  int max_pages, page_log2, num_pages, few_rows;
  int64_t max_new, max_len;  // what a sequence may hold (the launch is sized by them)
  int32_t* error_flag;
  // new rows of k and v, read from here while they are copied to their pages (null:
  // they are there)
  const void *k_new, *v_new;
  int64_t kn_st, kn_sh, vn_st, vn_sh;
  // the key axis in parts
  int splits;
  int64_t split_len;
  float *part_o, *part_ml;  // [splits][tokens * h_q][D], [splits][tokens * h_q][2]
  int64_t part_rows;
};

constexpr int kRows = 128;  // rows of a block of waves of their own

// A sequence of a paged batch: its query tokens [first, first + m) and keys.
struct Seq {
  int first, m, len;  // len: cached + m
};

__device__ __forceinline__ Seq paged_seq(const DenseParams& p, int b) {
  const int T = static_cast<int>(p.n_q);
  const int s0 = p.starts[b], s1 = p.starts[b + 1];
  const int c = p.cached[b];
  Seq s;
  s.first = min(max(s0, 0), T);
  s.m = max(min(s1, T) - s.first, 0);
  const int64_t cap = static_cast<int64_t>(p.max_pages) << p.page_log2;
  const int64_t len = static_cast<int64_t>(c) + s.m;
  const bool bad = s0 < 0 || s1 < s0 || s1 > T || c < 0 || len > cap || s.m > p.max_new || len > p.max_len;
  if (bad) {  // nothing of it is read or written
    if (p.error_flag != nullptr) atomicOr(p.error_flag, 1);
    s.m = 0;
  }
  s.len = bad ? 0 : c + s.m;
  return s;
}

enum View { kOne = 0, kTwo = 1 };  // (see the head of the file)

constexpr int kDrafts = 64;  // tokens of a sequence in a tree: an ancestor is a bit

// The keys a row sees: lo <= j < hi, a_lo <= j < a_hi, and new tokens cached + i for the bits i
// of kin.
struct Sees {
  int lo, hi, a_lo, a_hi, cached;
  uint64_t kin;
  __device__ __forceinline__ bool key(int j) const {
    const int i = j - cached;
    return (j >= lo && j < hi) || (j >= a_lo && j < a_hi) || (i >= 0 && i < kDrafts && (kin >> i & 1) != 0);
  }
  // some key of [x, y)
  __device__ __forceinline__ bool any(int x, int y) const {
    const int i = min(max(x - cached, 0), kDrafts), z = min(max(y - cached, 0), kDrafts);
    const uint64_t from = i < kDrafts ? ~uint64_t(0) << i : 0, to = z < kDrafts ? (uint64_t(1) << z) - 1 : ~uint64_t(0);
    return max(lo, x) < min(hi, y) || max(a_lo, x) < min(a_hi, y) || (kin & from & to) != 0;
  }
};

// The bits of 32 keys from the off-th new token on.
__device__ __forceinline__ uint32_t kin_word(uint64_t kin, int off) {
  if (off >= kDrafts || off <= -32) return 0u;
  return off >= 0 ? static_cast<uint32_t>(kin >> off) : static_cast<uint32_t>(kin) << -off;
}

// Lane i's new token of a sequence with m <= 64 of them: which new tokens it sees (itself and its
// ancestors; of those its window has left behind, the first keys only) and how many tokens
// above it (`depth`).  All lanes take part.  The ancestors meet by pointer doubling: after round r
// a lane knows the next 2^r of them.  A parent that does not come before its child is none.
__device__ __forceinline__ uint64_t draft_kin(const DenseParams& p, int first, int m, int cached, int& depth) {
  const int lane = threadIdx.x & 63;
  int up = -1;
  if (lane < m) {
    up = p.parents[first + lane];
    if (up < -1 || up >= lane) {
      if (p.error_flag != nullptr) atomicOr(p.error_flag, 1);
      up = -1;
    }
  }
  uint64_t kin = uint64_t(1) << lane;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int src = max(up, 0);
    const uint32_t a = static_cast<uint32_t>(__shfl(static_cast<int>(kin & 0xFFFFFFFFu), src, 64));
    const uint32_t b = static_cast<uint32_t>(__shfl(static_cast<int>(kin >> 32), src, 64));
    const int next = __shfl(up, src, 64);
    if (up >= 0) {
      kin |= static_cast<uint64_t>(b) << 32 | a;
      up = next;
    }
  }
  depth = __popcll(kin) - 1;
  if (p.window > 0 && depth >= p.window) {  // (ancestors by rising depth are its bits by rising index)
    const int keep = min(max(p.sinks - cached, 0), kDrafts);
    uint64_t rest = kin;
    for (int e = 0; e <= depth - p.window; ++e) {
      const uint64_t bit = rest & (~rest + 1);
      if (e >= keep) kin ^= bit;
      rest ^= bit;
    }
  }
  return kin;
}
__device__ __forceinline__ uint64_t lanes_kin(uint64_t kin, int src) {
  const uint32_t a = static_cast<uint32_t>(__shfl(static_cast<int>(kin & 0xFFFFFFFFu), src, 64));
  const uint32_t b = static_cast<uint32_t>(__shfl(static_cast<int>(kin >> 32), src, 64));
  return static_cast<uint64_t>(b) << 32 | a;
}

// What a row of a paged call at position pos sees; kin 0: a chain.
__device__ __forceinline__ Sees paged_sees(const DenseParams& p, int pos, int cached, uint64_t kin) {
  Sees s;
  s.lo = p.window > 0 ? max(pos + 1 - p.window, 0) : 0;
  s.hi = kin != 0 ? cached : pos + 1;
  s.a_lo = 0;
  s.a_hi = min(min(p.sinks, s.lo), s.hi);
  s.cached = cached;
  s.kin = kin;
  if (s.lo > s.hi) s.lo = s.hi;
  return s;
}

// Eight bits as the value they stand for before the scale.
__device__ __forceinline__ float code_value(uint8_t c, int e4m3) {
  return e4m3 ? __builtin_amdgcn_cvt_f32_fp8(c, 0) : static_cast<float>(static_cast<int8_t>(c));
}
// Four codes as floats.
template <bool E4M3>
__device__ __forceinline__ void code_floats(uint32_t w, float (&f)[4]) {
  if constexpr (E4M3) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int>(__builtin_amdgcn_sbfe(w, 8 * i, 8)));  // (one instruction a code)
  }
}
// The codes of 16 bytes of T, exact in bf16 too: eight (two words of them) or four.
template <typename T>
struct Codes;
template <>
struct Codes<uint16_t> {
  static __device__ __forceinline__ uint4 load(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, static_cast<int>(offset), 0, 0);
    return make_uint4(x.x, x.y, 0u, 0u);
  }
  static __device__ __forceinline__ uint4 load(const uint8_t* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    return make_uint4(x.x, x.y, 0u, 0u);
  }
  template <bool E4M3>
  static __device__ __forceinline__ uint4 widen(uint32_t x, uint32_t y) {
    if constexpr (E4M3) {  // (two codes an instruction)
      auto two = [](uint32_t w, auto high) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, decltype(high)::value));
      };
      const std::false_type lo;
      const std::true_type hi;
      return make_uint4(two(x, lo), two(x, hi), two(y, lo), two(y, hi));
    }
    float a[4], b[4];
    code_floats<E4M3>(x, a);
    code_floats<E4M3>(y, b);
    return make_uint4(Op<uint16_t>::pack2(a[0], a[1]), Op<uint16_t>::pack2(a[2], a[3]), Op<uint16_t>::pack2(b[0], b[1]),
                      Op<uint16_t>::pack2(b[2], b[3]));
  }
};
template <>
struct Codes<float> {
  static __device__ __forceinline__ uint4 load(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    return make_uint4(__builtin_amdgcn_raw_buffer_load_b32(r, static_cast<int>(offset), 0, 0), 0u, 0u, 0u);
  }
  static __device__ __forceinline__ uint4 load(const uint8_t* p) {
    return make_uint4(*reinterpret_cast<const uint32_t*>(p), 0u, 0u, 0u);
  }
  template <bool E4M3>
  static __device__ __forceinline__ uint4 widen(uint32_t x, uint32_t) {
    float a[4];
    code_floats<E4M3>(x, a);
    return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
  }
};
template <typename T>
__device__ __forceinline__ uint4 widen_one(const uint4& x, int e4m3) {
  return e4m3 ? Codes<T>::template widen<true>(x.x, x.y) : Codes<T>::template widen<false>(x.x, x.y);
}

// The row of key j: contiguous keys, or the sequence's pages (its new rows where the
// call brought them).  S is what the pages hold: T, or uint8_t for 8-bit codes, whose rows
// have a scale each.
template <typename T, bool PAGED, typename S = T>
struct KeyRows {
  const S *k, *v;
  const float *k_scale, *v_scale;
  int64_t ks_sb, ks_sn, vs_sb, vs_sn;
  int e4m3;
  int64_t k_sn, v_sn, k_sb, v_sb;
  const int32_t* table;
  int page_log2, page_mask, num_pages;
  int32_t* error_flag;
  const T *k_new, *v_new;  // row of key new_from
  int64_t kn_st, vn_st;
  int new_from;

  // The table's entry, to be checked where it is used: a check here would wait for it.
  __device__ __forceinline__ int entry_of(int j) const { return table[j >> page_log2]; }
  __device__ __forceinline__ int checked(int pg) const {
    if (static_cast<unsigned>(pg) < static_cast<unsigned>(num_pages)) return pg;
    if (error_flag != nullptr) atomicOr(error_flag, 1);
    return 0;
  }
  // The same for the tiles of a loop, behind which `report` says what was outside the pool (with a
  // check that sets the flag itself, 2048 tokens over 30720 of int8 take 1690 us for 1650).
  __device__ __forceinline__ int noted(int pg, int& outside) const {
    const bool in = static_cast<unsigned>(pg) < static_cast<unsigned>(num_pages);
    outside |= in ? 0 : 1;
    return in ? pg : 0;
  }
  __device__ __forceinline__ void report(int outside) const {
    if (outside != 0 && error_flag != nullptr) atomicOr(error_flag, 1);
  }
  // Pages of 8 bits: whether key j is one of the call's own rows, and where they are.
  __device__ __forceinline__ bool is_new(int j) const { return j >= new_from; }
  __device__ __forceinline__ void new_rows(int j, const T*& kr, const T*& vr) const {
    const int64_t x = j - new_from;
    kr = k_new + x * kn_st;
    vr = v_new + x * vn_st;
  }
  __device__ __forceinline__ void code_rows(int64_t pg, int j, const S*& kr, const S*& vr) const {
    const int64_t r = j & page_mask;
    kr = k + pg * k_sb + r * k_sn;
    vr = v + pg * v_sb + r * v_sn;
  }
  __device__ __forceinline__ float scale_of(bool of_v, int64_t pg, int j) const {
    const int64_t r = j & page_mask;
    return of_v ? v_scale[pg * vs_sb + r * vs_sn] : k_scale[pg * ks_sb + r * ks_sn];
  }
  __device__ __forceinline__ void in_page(int64_t pg, int j, const T*& kr, const T*& vr) const {
    const int64_t r = j & page_mask, x = j - new_from;
    const T *kp = k + pg * k_sb + r * k_sn, *vp = v + pg * v_sb + r * v_sn;
    kr = x >= 0 ? k_new + x * kn_st : kp;
    vr = x >= 0 ? v_new + x * vn_st : vp;
  }
  __device__ __forceinline__ void at(int j, const T*& kr, const T*& vr) const {
    if constexpr (PAGED) {
      in_page(checked(entry_of(j)), j, kr, vr);
    } else {
      kr = k + j * k_sn;
      vr = v + j * v_sn;
    }
  }
};

template <typename T, bool PAGED, typename S = T>
__device__ __forceinline__ KeyRows<T, PAGED, S> key_rows(const DenseParams& p, int b, int kvh, int first, int cached) {
  KeyRows<T, PAGED, S> r;
  const int64_t kb = PAGED ? 0 : b * p.k_sb, vb = PAGED ? 0 : b * p.v_sb;
  r.k = static_cast<const S*>(p.k) + kb + kvh * p.k_sh;
  r.v = static_cast<const S*>(p.v) + vb + kvh * p.v_sh;
  if constexpr (!std::is_same_v<S, T>) {
    r.k_scale = p.k_scale + kvh * p.ks_sh;
    r.v_scale = p.v_scale + kvh * p.vs_sh;
    r.ks_sb = p.ks_sb;
    r.ks_sn = p.ks_sn;
    r.vs_sb = p.vs_sb;
    r.vs_sn = p.vs_sn;
    r.e4m3 = p.e4m3;
  }
  r.k_sn = p.k_sn;
  r.v_sn = p.v_sn;
  r.k_sb = p.k_sb;
  r.v_sb = p.v_sb;
  r.table = PAGED ? p.table + b * p.table_stride : nullptr;
  r.page_log2 = p.page_log2;
  r.page_mask = (1 << p.page_log2) - 1;
  r.num_pages = p.num_pages;
  r.error_flag = p.error_flag;
  if constexpr (PAGED) {
    r.new_from = p.k_new != nullptr ? cached : 0x7FFFFFFF;
    r.k_new = static_cast<const T*>(p.k_new) + first * p.kn_st + kvh * p.kn_sh;
    r.v_new = static_cast<const T*>(p.v_new) + first * p.vn_st + kvh * p.vn_sh;
    r.kn_st = p.kn_st;
    r.vn_st = p.vn_st;
  }
  return r;
}

// q . k over d elements in fp32 (rows of 16 bytes).
template <typename T>
__device__ __forceinline__ float row_dot(const T* a, const T* b, int d) {
  float s = 0.0f;
  for (int e = 0; e < d; e += 8) s = Op<T>::dot(Op<T>::load(a + e), Op<T>::load(b + e), s);
  return s;
}

// A score (log2 units) of one pair.
template <typename T>
__device__ __forceinline__ float rule_of(const ScoreRule& r, float dot, float slope, int pos, int j) {
  const float dist = static_cast<float>(j - pos);
  if (sizeof(T) == 2 && r.cap == kSeries) return Rule<T, kFar>(r).z(r, dot, slope, dist);
  return Rule<T, kBias>(r).z(r, dot, slope, dist);
}

// One row by one wave, key by key, touching visible keys only.  Lane e holds
// features e, e + 64, ... of the (unnormalised) result o; m and l are the row's
// reference and sum.
template <typename T, bool PAGED>
__device__ __forceinline__ void exact_row(const KeyRows<T, PAGED>& rows, const ScoreRule& rule, const T* q, int d, int lo,
                                       int hi, float slope, int pos, float (&o)[4], float& m, float& l) {
  const int lane = threadIdx.x & 63;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = 0.0f;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = j0 + lane;
    const bool ok = j < hi;
    const T *kr, *vr;
    rows.at(ok ? j : lo, kr, vr);
    const float x = rule_of<T>(rule, row_dot(q, kr, d), slope, pos, j);
    const float top = wave_max(ok ? x : -INFINITY);
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
    const float a = exp2_w(m - ref);
    const float w = ok ? exp2_w(x - ref) : 0.0f;
    m = mn;
    l = l * a + wave_sum(w);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
    for (int t = 0; t < min(64, hi - j0); ++t) {
      const float wt = lane_value(w, t);
      const T *kt, *vt;
      rows.at(j0 + t, kt, vt);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < d) o[e] = fmaf(wt, ld(vt + lane + 64 * e), o[e]);
    }
  }
}

// exact_row for rows that see more than one interval: adds the keys of [x, y) that the row sees.
// depth: positions of drafted tokens behind the cached ones (null: a chain).
template <typename T, typename S, bool PAGED>
__device__ __forceinline__ void exact_keys(const KeyRows<T, PAGED, S>& rows, const ScoreRule& rule, const Sees& see, const T* q,
                                           int d, int x, int y, float slope, int pos, const int* depth, float (&o)[4],
                                           float& m, float& l) {
  constexpr bool HELD = !std::is_same_v<S, T>;
  const int lane = threadIdx.x & 63;
  for (int j0 = x; j0 < y; j0 += 64) {
    const int j = j0 + lane;
    const bool ok = j < y && see.key(j);
    float z = -INFINITY;
    if (ok) {
      const int at = depth != nullptr && j >= see.cached ? see.cached + depth[j - see.cached] : j;
      float dot = 0.0f;
      if (HELD && !rows.is_new(j)) {
        const S *kr, *vr;
        const int64_t pg = rows.checked(rows.entry_of(j));
        rows.code_rows(pg, j, kr, vr);
        if constexpr (HELD)
          for (int e = 0; e < d; ++e) dot = fmaf(ld(q + e), code_value(kr[e], rows.e4m3), dot);
        dot *= rows.scale_of(false, pg, j);
      } else {
        const T *kr, *vr;
        if constexpr (HELD)
          rows.new_rows(j, kr, vr);
        else
          rows.at(j, kr, vr);
        dot = row_dot(q, kr, d);
      }
      z = rule_of<T>(rule, dot, slope, pos, at);
    }
    uint64_t on = __ballot(ok);
    if (on == 0) continue;
    const float mn = fmaxf(m, wave_max(z)), ref = mn == -INFINITY ? 0.0f : mn;
    const float a = exp2_w(m - ref);
    const float w = ok ? exp2_w(z - ref) : 0.0f;
    m = mn;
    l = l * a + wave_sum(w);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
    while (on != 0) {
      const int t = __builtin_ctzll(on);
      on &= on - 1;
      float wt = lane_value(w, t);
      const int jt = j0 + t;
      if (HELD && !rows.is_new(jt)) {
        const S *kr, *vr;
        const int64_t pg = rows.checked(rows.entry_of(jt));
        rows.code_rows(pg, jt, kr, vr);
        wt *= rows.scale_of(true, pg, jt);
        if constexpr (HELD)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < d) o[e] = fmaf(wt, code_value(vr[lane + 64 * e], rows.e4m3), o[e]);
      } else {
        const T *kr, *vr;
        if constexpr (HELD)
          rows.new_rows(jt, kr, vr);
        else
          rows.at(jt, kr, vr);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lane + 64 * e < d) o[e] = fmaf(wt, ld(vr + lane + 64 * e), o[e]);
      }
    }
  }
}

// Which (sequence, tile of rows) a block of a ragged batch takes: the idx-th
// tile in sequence order, sequences with at most few_rows rows left out.
// Returns false past the last one.
__device__ __forceinline__ bool find_tile(const DenseParams& p, int idx, int block_rows, int& b, int& tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int t = 0;
    if (b0 + lane < p.batch) {
      const int64_t rows = static_cast<int64_t>(paged_seq(p, b0 + lane).m) * p.g;
      t = rows > p.few_rows ? static_cast<int>((rows + block_rows - 1) / block_rows) : 0;
    }
    const int incl = wave_incl_scan(t);
    const uint64_t past = __ballot(before + incl > idx);
    if (past != 0) {
      const int src = __builtin_ctzll(past);
      b = b0 + src;
      tile = idx - before - (lane_value(incl, src) - lane_value(t, src));
      return true;
    }
    before += lane_value(incl, 63);
  }
  return false;
}

// Rows of a block whose KW waves share each 32 rows and take the keys in turn.
constexpr int rows_of(int kw) { return kRows / kw; }

// Keys of a tile: 32 or 64 a wave.
template <typename T, int KW>
constexpr int key_tile() {
  return KW > 1 ? 32 * KW : (sizeof(T) == 2 ? 64 : 32);
}

// The most waves that may share rows: fp32 rows of 128 features fill the LDS with two.
template <typename T, int D>
constexpr int most_kw() {
  return sizeof(T) == 4 && D == 128 ? 2 : 4;
}

// Buffers of K and V in the LDS.  Two spare a barrier a tile, but where they leave a CU
// one block, two blocks of one buffer are the faster: each covers the other's waits
// (1024 x 2 causal rows of 8 / 2 heads, fp32, d = 64: 53 to 46 us).
template <typename T, int D, int KW>
constexpr int key_buffers() {
  return 4 * key_tile<T, KW>() * D * static_cast<int>(sizeof(T)) > 80 * 1024 ? 1 : 2;
}

// LDS of a block: the buffers, or at the end the waves' sums.
template <typename T, int D, int KW>
constexpr size_t rows_lds() {
  const size_t tiles = static_cast<size_t>(2) * key_buffers<T, D, KW>() * key_tile<T, KW>() * D * sizeof(T);
  const size_t sums = KW > 1 ? static_cast<size_t>(4) * 32 * (D + 4) * sizeof(float) : 0;
  return tiles > sums ? tiles : sums;
}

// Blocks on a CU: by LDS, and fp32 rows of 128 features want the registers of two.
template <typename T, int D, int KW>
constexpr int rows_per_cu() {
  return rows_lds<T, D, KW>() > 80 * 1024 || (sizeof(T) == 4 && D == 128) ? 1 : 2;
}

// The t-th tile to start, of tiles that get shorter under a causal mask, where `heads`
// blocks of each follow one another.  Longest first, blocks beyond those that run at
// once even the CUs out.  Where all run at once, two a CU, a CU would keep the t-th
// longest of each 256: the second 256 start shortest first (4096 causal rows of 16 / 4
// heads, d = 128, 512 blocks: 125 to 118 us; with 1008 blocks it costs 5%).
__device__ __forceinline__ int fold_tile(int t, int tiles, int heads) {
  const int per = heads < 256 ? 256 / heads : 1;
  const int round = t / per, at = t - round * per;
  if ((round & 1) == 0) return t;
  const int left = tiles - round * per;
  return round * per + (left < per ? left : per) - 1 - at;
}

// What a tile over pages of 8 bits holds: codes, or some of the call's own rows.  Each kind has a loop
// of its own in dense_rows; kAny: one loop for all, which asks of each tile.
enum { kGiven, kI8, kE4m3, kAny };

// Whether bf16 rows of 8-bit pages walk them in one loop: three of them with a rule of scores that takes
// many registers spill up to 183 of them.  2048 tokens over 30720, 32 / 8 heads, three loops and one:
//   d = 128, distance bias   2368 and 2358 us of int8, 2702 and 2266 of e4m3
//            far caps        2950 and 2631            3185 and 2582
//   d = 64, far caps         2220 and 2167            2156 and 2115
// (512 over 8192, d = 128, bias: 253 and 265, 299 and 258; d = 64, where nothing spills: 187 and 209, 183 and
// 206).  The other rules gain by three: plain scores, d = 128, 1694 to 1556 and 1546 to 1517.
template <typename T, int D, int RULE>
constexpr bool one_loop() {
  return sizeof(T) == 2 && (RULE == kFar || (RULE == kBias && D == 128));
}

// FRESH: tiles of a paged call's own rows are read as contiguous ones are.
template <typename T, int D, bool PAGED, int RULE, int KW, bool FRESH = false, int VIEW = kOne, typename S = T>
__device__ __forceinline__ void dense_rows(const DenseParams& p, const int w, char* lds) {
  constexpr bool SETS = VIEW == kTwo, HELD = !std::is_same_v<S, T>, TREE = SETS && PAGED;
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int RB = D * O::kEsize;      // bytes of a tile row
  constexpr int NCH = RB / 16;           // its chunks
  constexpr int E = 16 / O::kEsize;      // elements of a chunk
  constexpr int KT = key_tile<T, KW>();  // keys of a tile
  constexpr int NSUB = KT / (32 * KW), NC = D / 16, ND = D / 32;
  constexpr int RPP = kThreads / NCH;    // tile rows a pass of the block loads
  constexpr int NP = KT / RPP;
  constexpr int TB = KT * RB;            // bytes of a tile
  constexpr bool TWO = key_buffers<T, D, KW>() == 2;
  constexpr int BR = rows_of(KW);        // the block's rows
  constexpr int PS = D + 4;              // floats of a row of sums
  // lds: [2 buffers][K, V][TB], then [4 waves][32][PS]
  __shared__ int s_range[4][SETS ? 4 : 2];
  __shared__ float s_m[4][32], s_l[4][32];
  __shared__ int s_flag[4][32];
  __shared__ int s_depth[TREE ? kDrafts : 1];
  __shared__ __align__(16) float s_scale[HELD ? 4 : 1][HELD ? KT : 1];  // [buffer][K, V]

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave % KW, rw = wave / KW;
  const int nbh = PAGED ? p.h_kv : p.batch * p.h_kv;
  const int bh = w % nbh;
  int rest = w / nbh;
  const int split = rest % p.splits;
  rest /= p.splits;
  int b, kvh, tile, first = 0, m;
  int64_t n_keys;
  if constexpr (PAGED) {
    kvh = bh;
    if (!find_tile(p, rest, BR, b, tile)) return;
    const Seq s = paged_seq(p, b);
    first = s.first;
    m = s.m;
    n_keys = s.len;
    // the longest rows of a chunk first
    tile = (m * p.g + BR - 1) / BR - 1 - tile;
    if (tile < 0) return;
  } else {
    b = bh / p.h_kv;
    kvh = bh - b * p.h_kv;
    m = static_cast<int>(p.n_q);
    n_keys = p.n;
    const int tiles = static_cast<int>((p.n_q * p.g + BR - 1) / BR);
    const bool fold = rows_per_cu<T, D, KW>() == 2 && nbh * tiles * p.splits <= 512;
    tile = tiles - 1 - (fold ? fold_tile(rest, tiles, nbh * p.splits) : rest);
  }
  const KeyRows<T, PAGED, S> rows = key_rows<T, PAGED, S>(p, b, kvh, first, static_cast<int>(n_keys) - m);

  // this lane's row
  const int r = tile * BR + rw * 32 + (lane & 31);
  const bool real = r < m * p.g;
  const int tok = real ? r / p.g : 0;
  const int hq = kvh * p.g + (real ? r - tok * p.g : 0);
  int pos = PAGED ? static_cast<int>(n_keys) - m + tok : static_cast<int>(p.q_pos0) + tok;
  const int cached = PAGED ? static_cast<int>(n_keys) - m : 0;
  const bool tree = TREE && p.parents != nullptr;
  int lo = 0, hi = 0;
  Sees see{0, 0, 0, 0, cached, 0};
  int b_lo = 0, b_hi = 0;  // of the second range of tiles: lo and hi, or from there to the drafts' end
  if constexpr (TREE) {
    uint64_t kin = 0;
    if (tree) {
      int depth;
      const uint64_t all = draft_kin(p, first, m, cached, depth);
      if (lane < kDrafts) s_depth[lane] = depth;  // (each wave the same)
      kin = lanes_kin(all, tok);
      pos = cached + __shfl(depth, tok, 64);
    }
    if (real) {
      see = paged_sees(p, pos, cached, kin);
      lo = see.lo;
      hi = see.hi;
      b_lo = lo;
      b_hi = tree ? static_cast<int>(n_keys) : hi;
    }
  } else if constexpr (SETS) {
    if (real) {
      const int4 s = reinterpret_cast<const int4*>(p.spans)[b * p.n_q + tok];
      lo = max(s.x, 0);
      hi = static_cast<int>(min(static_cast<int64_t>(s.y), n_keys));
      if (hi <= lo) lo = hi = 0;
      int x = max(s.z, 0), y = static_cast<int>(min(static_cast<int64_t>(s.w), n_keys));
      if (y <= x) x = y = 0;
      if (hi == lo) {  // (one interval is the second one)
        lo = x;
        hi = y;
        x = y = 0;
      }
      see = Sees{lo, hi, x, y, static_cast<int>(n_keys), 0};
      b_lo = lo;
      b_hi = hi;
    }
  } else if (real) {
    if (!PAGED && p.spans != nullptr) {
      const int2 s = p.spans[b * p.n_q + tok];
      lo = max(s.x, 0);
      hi = static_cast<int>(min(static_cast<int64_t>(s.y), n_keys));
    } else {
      hi = static_cast<int>(min(static_cast<int64_t>(pos) + 1, n_keys));
    }
    if (hi <= lo) lo = hi = 0;
  }
  const bool some = real && (SETS ? b_hi > b_lo : hi > lo);
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const int lo_min = wave_min_i(some ? (SETS ? b_lo : lo) : 0x7FFFFFFF), hi_max = wave_max_i(some ? (SETS ? b_hi : hi) : 0);
  int a_min = 0x7FFFFFFF, a_max = 0;
  if constexpr (SETS) {
    const bool has = real && see.a_hi > see.a_lo;
    a_min = wave_min_i(has ? see.a_lo : 0x7FFFFFFF);
    a_max = wave_max_i(has ? see.a_hi : 0);
  }
  const int lo_max = wave_max_i(real ? lo : 0), hi_min = wave_min_i(real ? hi : 0x7FFFFFFF);
  if (lane == 0) {
    s_range[wave][0] = lo_min;
    s_range[wave][1] = hi_max;
    if constexpr (SETS) {
      s_range[wave][2] = a_min;
      s_range[wave][3] = a_max;
    }
  }
  const T* qrow = static_cast<const T*>(p.q) + (PAGED ? first * p.q_sn : b * p.q_sb) + tok * p.q_sn + hq * p.q_sh;
  Frag qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = 16 * c + 8 * half;
    qf[c] = real && e < p.d ? O::load(qrow + e) : O::zero();
  }
  __syncthreads();
  int k_lo = __builtin_amdgcn_readfirstlane(min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0])));
  int k_hi = __builtin_amdgcn_readfirstlane(max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1])));
  int part_lo = 0, part_hi = 0x7FFFFFFF;
  int first_a = 0;             // keys below it are seen by some row, others from k_lo on
  Tiles walk{0, 0, 0, 0};      // kTwo: the block's tiles, of which it takes nt from t0 on
  int part_x[2] = {0, 0}, part_y[2] = {0, 0};  // their keys
  if constexpr (SETS) {
    const int a_lo = __builtin_amdgcn_readfirstlane(min(min(s_range[0][2], s_range[1][2]), min(s_range[2][2], s_range[3][2])));
    first_a = __builtin_amdgcn_readfirstlane(max(max(s_range[0][3], s_range[1][3]), max(s_range[2][3], s_range[3][3])));
    walk = first_a > a_lo ? tiles_of(a_lo, first_a, k_hi > k_lo ? k_lo : 0, k_hi, KT) : tiles_of(0, 0, k_hi > k_lo ? k_lo : 0, k_hi, KT);
  } else if (p.splits > 1) {
    const int64_t s0 = split * p.split_len, s1 = s0 + p.split_len;
    part_lo = static_cast<int>(min(s0, static_cast<int64_t>(0x7FFFFFFF)));
    part_hi = static_cast<int>(min(s1, static_cast<int64_t>(0x7FFFFFFF)));
    k_lo = max(k_lo, part_lo);
    k_hi = min(k_hi, part_hi);
  }
  int t0, nt;
  if constexpr (SETS) {
    // parts are equal shares of the block's tiles; over pages as long as each other (p.split_len keys),
    // so that short sequences have few
    const int per = TREE ? (p.splits > 1 ? static_cast<int>(p.split_len / KT) : walk.n) : (walk.n + p.splits - 1) / p.splits;
    t0 = static_cast<int>(min(static_cast<int64_t>(split) * per, static_cast<int64_t>(walk.n)));
    nt = min(per, walk.n - t0);
    if (p.splits > 1 && nt == 0) {  // (a part without a key: the join wants its sums alone)
      const int64_t at = (PAGED ? first : static_cast<int64_t>(b) * p.n_q) + tok;
      if (real && half == 0 && kw == 0)
        *reinterpret_cast<float2*>(p.part_ml + (split * p.part_rows + at * p.h_q + hq) * 2) = make_float2(-INFINITY, 0.0f);
      return;
    }
    part_x[0] = (walk.x0 + min(t0, walk.n1)) * KT;
    part_y[0] = (walk.x0 + min(t0 + nt, walk.n1)) * KT;
    part_x[1] = (walk.y0 + max(t0 - walk.n1, 0)) * KT;
    part_y[1] = (walk.y0 + max(t0 + nt - walk.n1, 0)) * KT;
  } else {
    t0 = k_lo / KT;
    nt = k_hi > k_lo ? (k_hi + KT - 1) / KT - t0 : 0;
  }
  // the first key of the t-th tile; where a key is looked up, one that some row sees
  auto tile_key = [&](int t) { return SETS ? walk.at(t0 + t) * KT : (t0 + t) * KT; };
  auto seen_key = [&](int j) { return TREE && j >= first_a ? max(j, k_lo) : j; };

  // staging: chunk sc of tile rows sr, sr + RPP, ....  Of paged keys, a wave's rows of
  // a load lie in one page, looked up a tile before; tiles that reach past the pages'
  // keys (the call's own rows unless FRESH, a tile of both, the end) take each row's
  // address.
  const int sc = tid % NCH, sr = tid / NCH;
  const bool chunk_ok = sc * E < p.d;
  const int last = static_cast<int>(n_keys) - 1;
  const int64_t kst = rows.k_sn * O::kEsize, vst = rows.v_sn * O::kEsize;  // bytes of a row
  const uint32_t ks = static_cast<uint32_t>(kst), vs = static_cast<uint32_t>(vst);
  const int my = PAGED ? lane / NCH : sr;
  const uint32_t koff = chunk_ok ? my * ks + sc * 16 : kNoChunk, voff = chunk_ok ? my * vs + sc * 16 : kNoChunk;
  uint4 kreg[NP], vreg[NP];
  int pg[PAGED ? NP : 1];
  // HELD: the scale that this thread fetches, of key `scale_key` of a tile (K's by SW waves, V's by the
  // next), and its page
  constexpr int SW = KT > 64 ? KT / 64 : 1;
  const int scale_key = KT < 64 ? lane : tid & (KT - 1);
  const bool scale_here = wave < 2 * SW && (KT >= 64 || lane < KT), scale_of_v = wave >= SW;
  const uint32_t ks8 = static_cast<uint32_t>(rows.k_sn), vs8 = static_cast<uint32_t>(rows.v_sn);
  const uint32_t koff8 = chunk_ok ? my * ks8 + sc * E : kNoChunk, voff8 = chunk_ok ? my * vs8 + sc * E : kNoChunk;
  int scale_pg = 0;
  float scale_reg = 1.0f;
  int outside = 0;  // whether a page of a tile was outside the pool
  [[maybe_unused]] bool as_codes = false;  // kAny: whether the loaded tile is of codes alone
  const int paged_end = PAGED ? min(rows.new_from, static_cast<int>(n_keys)) : 0;
  constexpr int RPW = 64 / NCH;  // rows of a wave's load
  auto find_pages = [&](int t) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < NP; ++i) pg[i] = rows.entry_of(min(seen_key(tile_key(t) + i * RPP + wave * RPW), last));
      if (HELD && scale_here) scale_pg = rows.entry_of(min(seen_key(tile_key(t) + scale_key), last));
    }
  };
  // (kind: of HELD tiles whether they are codes alone, int8 or e4m3, or have the call's own rows)
  auto load_tile = [&](auto kind, int t) {
    constexpr int KIND = decltype(kind)::value;
    const int j0 = tile_key(t);
    if constexpr (HELD) {
      const int j = min(seen_key(j0 + scale_key), last);
      scale_reg = 1.0f;
      if (scale_here && !rows.is_new(j)) scale_reg = rows.scale_of(scale_of_v, rows.noted(scale_pg, outside), j);
      if (KIND == kAny) as_codes = j0 + KT <= paged_end;
      if (KIND == kAny ? as_codes : KIND != kGiven) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int64_t page = rows.noted(__builtin_amdgcn_readfirstlane(pg[i]), outside), r0 = (j0 + i * RPP + wave * RPW) & rows.page_mask;
          kreg[i] = Codes<T>::load(row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes), koff8);
          vreg[i] = Codes<T>::load(row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes), voff8);
        }
        return;
      }
      if (j0 < rows.new_from) {  // a tile of both
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int x = min(seen_key(j0 + sr + i * RPP), last);
          kreg[i] = vreg[i] = make_uint4(0u, 0u, 0u, 0u);
          if (!chunk_ok) continue;
          if (rows.is_new(x)) {
            const T *kr, *vr;
            rows.new_rows(x, kr, vr);
            kreg[i] = *reinterpret_cast<const uint4*>(kr + sc * E);
            vreg[i] = *reinterpret_cast<const uint4*>(vr + sc * E);
          } else {
            const S *kr, *vr;
            rows.code_rows(rows.noted(rows.entry_of(x), outside), x, kr, vr);
            kreg[i] = widen_one<T>(Codes<T>::load(kr + sc * E), rows.e4m3);
            vreg[i] = widen_one<T>(Codes<T>::load(vr + sc * E), rows.e4m3);
          }
        }
        return;
      }
    }
    if constexpr (PAGED) {
      if (!HELD && j0 + KT <= paged_end) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int64_t page = rows.noted(__builtin_amdgcn_readfirstlane(pg[i]), outside), r0 = (j0 + i * RPP + wave * RPW) & rows.page_mask;
          kreg[i] = row_load(row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes), koff);
          vreg[i] = row_load(row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes), voff);
        }
      } else if (HELD || (FRESH && j0 >= rows.new_from)) {
        const int left = static_cast<int>(n_keys) - j0, x = j0 - rows.new_from, db = p.d * O::kEsize;
        const uint32_t kn = static_cast<uint32_t>(rows.kn_st * O::kEsize), vn = static_cast<uint32_t>(rows.vn_st * O::kEsize);
        const auto kb = row_buffer(rows.k_new + x * rows.kn_st, left >= KT ? kAllBytes : static_cast<int>((left - 1) * kn) + db);
        const auto vb = row_buffer(rows.v_new + x * rows.vn_st, left >= KT ? kAllBytes : static_cast<int>((left - 1) * vn) + db);
        const uint32_t r = in_branch(sr), ko = chunk_ok ? r * kn + sc * 16 : kNoChunk, vo = chunk_ok ? r * vn + sc * 16 : kNoChunk;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          kreg[i] = row_load(kb, ko + i * RPP * kn);
          vreg[i] = row_load(vb, vo + i * RPP * vn);
        }
      } else if constexpr (!HELD) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const T *kr, *vr;
          rows.at(min(seen_key(j0 + sr + i * RPP), last), kr, vr);
          kreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(kr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
          vreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(vr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
        }
      }
    } else {
      const int left = static_cast<int>(n_keys) - j0;  // at least one
      const int db = p.d * O::kEsize;
      const auto kb = row_buffer(rows.k + j0 * rows.k_sn, left >= KT ? kAllBytes : static_cast<int>((left - 1) * kst) + db);
      const auto vb = row_buffer(rows.v + j0 * rows.v_sn, left >= KT ? kAllBytes : static_cast<int>((left - 1) * vst) + db);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        kreg[i] = row_load(kb, koff + i * RPP * ks);
        vreg[i] = row_load(vb, voff + i * RPP * vs);
      }
    }
  };
  auto store_tile = [&](auto kind, int buf) {
    constexpr int KIND = decltype(kind)::value;
    char* kt = lds + buf * 2 * TB;
    if constexpr (HELD) {
      if (scale_here) s_scale[2 * buf + (scale_of_v ? 1 : 0)][scale_key] = scale_reg;
      auto widened = [&](auto e4m3) {
        constexpr bool E4M3 = decltype(e4m3)::value;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int at = chunk_at<RB>(sr + i * RPP, sc);
          *reinterpret_cast<uint4*>(kt + at) = Codes<T>::template widen<E4M3>(kreg[i].x, kreg[i].y);
          *reinterpret_cast<uint4*>(kt + TB + at) = Codes<T>::template widen<E4M3>(vreg[i].x, vreg[i].y);
        }
      };
      if (KIND == kAny ? as_codes : KIND != kGiven) {
        if (KIND == kE4m3 || (KIND == kAny && rows.e4m3))
          widened(std::true_type());
        else
          widened(std::false_type());
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = chunk_at<RB>(sr + i * RPP, sc);
      *reinterpret_cast<uint4*>(kt + at) = kreg[i];
      *reinterpret_cast<uint4*>(kt + TB + at) = vreg[i];
    }
  };

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{};
  float mref = -INFINITY, lsum = 0.0f;

  auto walk_tiles = [&](auto kind, const int from, const int to) {
    if (to > from) {
      find_pages(from);
      load_tile(kind, from);
      if (to > from + 1) find_pages(from + 1);
      store_tile(kind, TWO ? from & 1 : 0);
    }
    settle(qf);
    for (int t = from; t < to; ++t) {
      __syncthreads();
      if (t + 1 < to) load_tile(kind, t + 1);
      if (t + 2 < to) find_pages(t + 2);
      const int k0 = tile_key(t) + kw * 32 * NSUB;
      if ((k0 < hi_max && k0 + 32 * NSUB > lo_min) || (SETS && k0 < a_max && k0 + 32 * NSUB > a_min)) {
        const char* kt = lds + (TWO ? (t & 1) * 2 * TB : 0) + kw * 32 * NSUB * RB;
        const char* vt = kt + TB;
        f32x16 s[NSUB];
#pragma unroll
        for (int u = 0; u < NSUB; ++u) s[u] = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int u = 0; u < NSUB; ++u) s[u] = O::mfma(O::template row_frag<RB>(kt, 32 * u, c, lane), qf[c], s[u]);

        const int kl = k0 + 4 * half;  // key of register 0
        const float dist = static_cast<float>(kl - pos);
        [[maybe_unused]] const float* ksc = s_scale[HELD && TWO ? 2 * (t & 1) : 0] + (HELD ? kw * 32 * NSUB + 4 * half : 0);
        [[maybe_unused]] const float* vsc = s_scale[HELD && TWO ? 2 * (t & 1) + 1 : (HELD ? 1 : 0)] + (HELD ? kw * 32 * NSUB + 4 * half : 0);
        if constexpr (HELD)
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 x = *reinterpret_cast<const float4*>(ksc + 32 * u + 8 * e);
              s[u][4 * e] *= x.x;
              s[u][4 * e + 1] *= x.y;
              s[u][4 * e + 2] *= x.z;
              s[u][4 * e + 3] *= x.w;
            }
        if (TREE && has_bias(RULE) && tree && k0 + 32 * NSUB > cached) {  // (drafts lie at cached + depth)
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int j = kl + 32 * u + 8 * (i >> 2) + (i & 3), x = j - cached;
              const int at = x < 0 ? j : cached + s_depth[TREE ? min(x, kDrafts - 1) : 0];
              s[u][i] = rule.z(p.rule, s[u][i], slope, static_cast<float>(at - pos));
            }
        } else {
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              s[u][i] = rule.z(p.rule, s[u][i], slope, dist + static_cast<float>(32 * u + 8 * (i >> 2) + (i & 3)));
        }
        const bool whole = k0 >= lo_max && k0 + 32 * NSUB <= hi_min && (SETS || (k0 >= part_lo && k0 + 32 * NSUB <= part_hi));
        if (SETS && !whole) {
          const int a = in_branch(lo - kl), z = in_branch(hi - kl), x = in_branch(see.a_lo - kl), y = in_branch(see.a_hi - kl);
#pragma unroll
          for (int u = 0; u < NSUB; ++u) {
            const uint32_t kin = TREE ? kin_word(see.kin, k0 + 32 * u - cached) >> (4 * half) : 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int jj = 8 * (i >> 2) + (i & 3), j = 32 * u + jj;
              const bool sees = (j >= a && j < z) || (j >= x && j < y) || (TREE && (kin >> jj & 1u) != 0);
              if (!sees) s[u][i] = Rule<T, RULE>::kHidden;
            }
          }
        } else if (!whole) {
          const int a = in_branch(max(lo, part_lo) - kl), z = in_branch(min(hi, part_hi) - kl);
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int j = 32 * u + 8 * (i >> 2) + (i & 3);
              if (j < a || j >= z) s[u][i] = Rule<T, RULE>::kHidden;
            }
        }
        float top = Rule<T, RULE>::kHidden;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = rule.better(top, s[u][i]);
        top = fmaf(rule.better(top, other_half(top)), rule.a, rule.b);
        if (__ballot(top > mref + 8.0f) != 0) {
          const float mn = fmaxf(mref, top);
          const float alpha = mref == mn ? 1.0f : exp2_w(mref - mn);
          mref = mn;
          lsum *= alpha;
#pragma unroll
          for (int i = 0; i < ND; ++i) acc[i] *= alpha;
        }
        const float nref = rule.b - (mref == -INFINITY ? 0.0f : mref);
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[u][i] = exp2_w(fmaf(s[u][i], rule.a, nref));
            lsum += s[u][i];
          }
        if constexpr (HELD)
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 x = *reinterpret_cast<const float4*>(vsc + 32 * u + 8 * e);
              s[u][4 * e] *= x.x;
              s[u][4 * e + 1] *= x.y;
              s[u][4 * e + 2] *= x.z;
              s[u][4 * e + 3] *= x.w;
            }
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const Frag pf = O::pack(s[u], c);
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] = O::mfma(O::template col_frag<RB>(vt, 32 * u + 16 * c, 32 * i, lane), pf, acc[i]);
          }
      }
      if constexpr (!TWO) __syncthreads();
      if (t + 1 < to) store_tile(kind, TWO ? (t + 1) & 1 : 0);
    }
  };
  if constexpr (HELD && one_loop<T, D, RULE>()) {
    walk_tiles(std::integral_constant<int, kAny>(), 0, nt);
  } else if constexpr (HELD) {
    int held = nt;  // the tiles of codes alone, which come first
    while (held > 0 && tile_key(held - 1) + KT > paged_end) --held;
    if (rows.e4m3)
      walk_tiles(std::integral_constant<int, kE4m3>(), 0, held);
    else
      walk_tiles(std::integral_constant<int, kI8>(), 0, held);
    walk_tiles(std::integral_constant<int, kGiven>(), held, nt);
  } else {
    walk_tiles(std::integral_constant<int, kGiven>(), 0, nt);
  }

  if constexpr (PAGED) rows.report(outside);

  // the row's sums, joined over the half-waves (they share the reference)
  lsum += other_half(lsum);
  float worst = finite(lsum) ? 0.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) worst = finite(acc[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, other_half(worst));
  // Where a row's results go: the output, or its part.
  const int64_t out0 = PAGED ? first * p.o_sn : b * p.o_sb;
  const int64_t row0 = PAGED ? first : static_cast<int64_t>(b) * p.n_q;
  auto put = [&](int tk, int h, int dd, float a, float c, float e, float f) {  // four features, normalised unless in parts
    if (p.splits > 1) {
      *reinterpret_cast<float4*>(p.part_o + (split * p.part_rows + (row0 + tk) * p.h_q + h) * D + dd) = make_float4(a, c, e, f);
    } else {
      const int64_t at = out0 + tk * p.o_sn + h * p.o_sh + dd;
      O::store4(static_cast<T*>(p.out) + at, a, c, e, f);
      if (p.out_low != nullptr) O::store4(static_cast<T*>(p.out_low) + at, O::left(a), O::left(c), O::left(e), O::left(f));
    }
  };
  auto put_sums = [&](int tk, int h, float mm, float l, bool any, bool here) {
    if (p.splits > 1) {
      // (a part whose visible keys all scored -inf says so by a finite m)
      float* pml = p.part_ml + (split * p.part_rows + (row0 + tk) * p.h_q + h) * 2;
      pml[0] = here && mm == -INFINITY ? -3.0e38f : mm;
      pml[1] = l;
    } else if (p.lse != nullptr) {
      p.lse[(static_cast<int64_t>(b) * p.h_q + h) * p.n_q + tk] = any ? mm + __log2f(l) : INFINITY;
    }
  };
  bool here;
  if constexpr (SETS)
    here = real && (see.any(part_x[0], part_y[0]) || see.any(part_x[1], part_y[1]));
  else
    here = some && max(lo, part_lo) < min(hi, part_hi);
  // no key: zeros, whatever hidden values its tiles' sums met; only keys of score -inf: NaN,
  // as a softmax of them is
  if constexpr (KW == 1) {
    const bool again = some && worst != 0.0f;
    if (real && !again) {
      const float inv = p.splits > 1 ? 1.0f : 1.0f / lsum;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dd = 32 * i + 8 * e + 4 * half;
          if (dd < p.d)
            put(tok, hq, dd, some ? acc[i][4 * e] * inv : 0.0f, some ? acc[i][4 * e + 1] * inv : 0.0f,
                some ? acc[i][4 * e + 2] * inv : 0.0f, some ? acc[i][4 * e + 3] * inv : 0.0f);
        }
      if (half == 0) put_sums(tok, hq, mref, lsum, some, here);
    }
    worst = again ? 1.0f : 0.0f;
  } else {
    if (half == 0) {
      s_m[wave][lane] = mref;
      s_l[wave][lane] = lsum;
      s_flag[wave][lane] = (some && worst != 0.0f ? 1 : 0) | (some ? 2 : 0) | (here ? 4 : 0);
    }
    __syncthreads();  // every wave is past its tiles: their LDS holds the sums now
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(sums + (wave * 32 + (lane & 31)) * PS + 32 * i + 8 * e + 4 * half) =
            make_float4(acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]);
    __syncthreads();
    for (int x = tid; x < BR * (D / 4); x += kThreads) {
      const int rr = x / (D / 4), dd = (x - rr * (D / 4)) * 4, wv = rr / 32 * KW, ln = rr & 31;
      const int rx = tile * BR + rr;
      if (dd >= p.d || rx >= m * p.g) continue;
      int flag = 0;
      float mm = -INFINITY;
#pragma unroll
      for (int y = 0; y < KW; ++y) {
        flag |= s_flag[wv + y][ln];
        mm = fmaxf(mm, s_m[wv + y][ln]);
      }
      if (flag & 1) continue;
      const float ref = mm == -INFINITY ? 0.0f : mm;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.0f;
#pragma unroll
      for (int y = 0; y < KW; ++y) {
        const float a = exp2_w(s_m[wv + y][ln] - ref);
        const float4 v = *reinterpret_cast<const float4*>(sums + ((wv + y) * 32 + ln) * PS + dd);
        l = fmaf(a, s_l[wv + y][ln], l);
        o.x = fmaf(a, v.x, o.x);
        o.y = fmaf(a, v.y, o.y);
        o.z = fmaf(a, v.z, o.z);
        o.w = fmaf(a, v.w, o.w);
      }
      const int tk = rx / p.g, h = kvh * p.g + rx - tk * p.g;
      const float inv = p.splits > 1 ? 1.0f : 1.0f / l;
      const bool any = (flag & 2) != 0;
      put(tk, h, dd, any ? o.x * inv : 0.0f, any ? o.y * inv : 0.0f, any ? o.z * inv : 0.0f, any ? o.w * inv : 0.0f);
      if (dd == 0) put_sums(tk, h, mm, l, any, (flag & 4) != 0);
    }
    int bad = 0;
#pragma unroll
    for (int y = 0; y < KW; ++y) bad |= s_flag[rw * KW + y][lane & 31] & 1;
    worst = bad && (lane & (KW - 1)) == kw ? 1.0f : 0.0f;  // shared out among the waves
  }

  uint64_t todo = __ballot(worst != 0.0f && half == 0);
  while (todo != 0) {  // rows to compute again, one after the other by a whole wave
    const int src = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int a = max(lane_value(lo, src), part_lo), z = min(lane_value(hi, src), part_hi);
    const int ps = lane_value(pos, src), tk = lane_value(tok, src), h = lane_value(hq, src);
    const float sl = lane_value(slope, src);
    float o[4], mm, ll;
    bool keys = a < z;
    const T* qr = static_cast<const T*>(p.q) + (PAGED ? first * p.q_sn : b * p.q_sb) + tk * p.q_sn + h * p.q_sh;
    if constexpr (SETS) {
      const uint32_t k0 = lane_value(static_cast<int>(see.kin & 0xFFFFFFFFu), src), k1 = lane_value(static_cast<int>(see.kin >> 32), src);
      const Sees row{lane_value(lo, src), lane_value(hi, src), lane_value(see.a_lo, src), lane_value(see.a_hi, src), see.cached,
                     static_cast<uint64_t>(k1) << 32 | k0};
      mm = -INFINITY;
      ll = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        exact_keys<T, S, PAGED>(rows, p.rule, row, qr, p.d, part_x[x], min(part_y[x], static_cast<int>(n_keys)), sl, ps,
                                tree ? s_depth : nullptr, o, mm, ll);
      keys = row.any(part_x[0], part_y[0]) || row.any(part_x[1], part_y[1]);
    } else {
      exact_row<T, PAGED>(rows, p.rule, qr, p.d, a, z, sl, ps, o, mm, ll);
    }
    const float inv = 1.0f / ll;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dd = lane + 64 * e;
      if (dd >= p.d) continue;
      if (p.splits > 1) {
        p.part_o[(split * p.part_rows + (row0 + tk) * p.h_q + h) * D + dd] = o[e];
      } else {
        const int64_t at = out0 + tk * p.o_sn + h * p.o_sh + dd;
        O::store1(static_cast<T*>(p.out) + at, o[e] * inv);
        if (p.out_low != nullptr) O::store1(static_cast<T*>(p.out_low) + at, O::left(o[e] * inv));
      }
    }
    if (lane == 0) put_sums(tk, h, mm, ll, true, keys);
  }
}

// Joins the parts of a row, by one wave.  A part without a key has m = -inf and
// l = 0 and its o is not read.
template <typename T, int D>
__device__ __forceinline__ void dense_join(const DenseParams& p, const int64_t row) {
  const int lane = threadIdx.x & 63;
  if (row >= p.part_rows) return;
  const int64_t tok = row / p.h_q, hq = row - tok * p.h_q;
  const int64_t b = p.starts != nullptr ? 0 : tok / p.n_q, t = tok - b * p.n_q;
  if (p.starts != nullptr) {  // a row behind the last sequence, or of one that is refused, stays as it was
    bool mine = false;
    for (int s0 = 0; s0 < p.batch; s0 += 64) {
      bool in = false;
      if (s0 + lane < p.batch) {
        const Seq s = paged_seq(p, s0 + lane);
        in = t >= s.first && t < s.first + s.m && static_cast<int64_t>(s.m) * p.g > p.few_rows;
      }
      mine |= __ballot(in) != 0;
    }
    if (!mine) return;
  }
  constexpr int L = D / 64;  // features of a lane: lane * L ..
  float m = -INFINITY, l = 0.0f, o[L];
  bool seen = false;
#pragma unroll
  for (int e = 0; e < L; ++e) o[e] = 0.0f;
  for (int s0 = 0; s0 < p.splits; s0 += 4) {  // four parts' loads in flight
    float2 ml[4];
    float v[4][L];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = min(s0 + i, p.splits - 1) * p.part_rows + row;
      ml[i] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
#pragma unroll
      for (int e = 0; e < L; ++e) v[i][e] = p.part_o[at * D + lane * L + e];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i >= p.splits) continue;
      seen |= ml[i].x != -INFINITY;
      if (ml[i].y == 0.0f) continue;  // (an empty part: its o was not written)
      const float mn = fmaxf(m, ml[i].x), ref = mn == -INFINITY ? 0.0f : mn;
      const float a = exp2_w(m - ref), w = exp2_w(ml[i].x - ref);
      m = mn;
      l = fmaf(l, a, ml[i].y * w);
#pragma unroll
      for (int e = 0; e < L; ++e) o[e] = fmaf(v[i][e], w, o[e] * a);
    }
  }
  T* orow = static_cast<T*>(p.out) + b * p.o_sb + t * p.o_sn + hq * p.o_sh;
  // no key: zeros; only keys of score -inf: NaN
  const float inv = seen ? 1.0f / l : 0.0f;
#pragma unroll
  for (int e = 0; e < L; ++e)
    if (lane * L + e < p.d) {
      Op<T>::store1(orow + lane * L + e, o[e] * inv);
      if (p.out_low != nullptr)
        Op<T>::store1(static_cast<T*>(p.out_low) + (orow - static_cast<T*>(p.out)) + lane * L + e, Op<T>::left(o[e] * inv));
    }
  if (p.lse != nullptr && lane == 0) p.lse[(b * p.h_q + hq) * p.n_q + t] = seen ? m + __log2f(l) : INFINITY;
}

}  // namespace tile
}  // namespace ssa
