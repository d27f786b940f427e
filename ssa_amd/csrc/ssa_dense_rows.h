// Softmax attention of many query rows over contiguous or paged keys: the
// forward kernel of ssa_masked_attention and of ssa_paged_step's chunks.
//
//   o_i = sum_j p_ij v_j,  p = softmax over lo_i <= j < hi_i of the score rule
//
// A block of four waves takes 128 rows of one KV head: a row is a (token, query
// head of the group) pair, tokens first, so that the g heads that share a key
// read its tile once and a causal block's diagonal is 128 / g tokens wide.  Each
// wave keeps 32 rows: Q as B operands in registers, S^T = K Q^T with one row's
// scores down a lane's registers (the running maximum and sum need one exchange
// with the other half-wave), P^T as the B operand of O^T += V^T P^T without
// leaving its registers (ssa_tile.h).  K and V tiles of 64 keys (32 in fp32)
// pass through a double LDS buffer, the next tile's global loads in flight
// meanwhile.  Tiles that no row of a wave sees are skipped, tiles that every row
// sees whole take no mask arithmetic.
//
// The running reference m is only moved when a tile's maximum exceeds it by more
// than 8 (in log2): weights then reach 2^8, which costs fp32 sums and bf16
// weights no relative precision, and most tiles rescale nothing.
//
// A masked key's weight is 0, but 0 times an infinity or NaN in its value row is
// not: a row whose accumulators end up other than finite is computed again key
// by key (exact_row), reading visible keys only.
#pragma once

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
  const int2* spans;  // null: causal by position
  ScoreRule rule;
  // paged: k and v are the pools [pages][page rows][h_kv][d] (sb = page stride)
  const int32_t *table, *starts, *cached;
  int64_t table_stride;
  int max_pages, page_log2, num_pages, few_rows;
  int64_t max_new, max_len;  // what a sequence may hold (the launch is sized by them)
  int32_t* error_flag;
  // the key axis in parts
  int splits;
  int64_t split_len;
  float *part_o, *part_ml;  // [splits][tokens * h_q][D], [splits][tokens * h_q][2]
  int64_t part_rows;
};

constexpr int kRows = 128;  // rows of a block

template <typename T>
constexpr int key_tile() {
  return sizeof(T) == 2 ? 64 : 32;
}

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

// The row of key j: contiguous keys, or the sequence's pages.
template <typename T, bool PAGED>
struct KeyRows {
  const T *k, *v;
  int64_t k_sn, v_sn, k_sb, v_sb;
  const int32_t* table;
  int page_log2, page_mask, num_pages;
  int32_t* error_flag;

  __device__ __forceinline__ int page_of(int j) const {
    int pg = table[j >> page_log2];
    if (static_cast<unsigned>(pg) >= static_cast<unsigned>(num_pages)) {
      if (error_flag != nullptr) atomicOr(error_flag, 1);
      pg = 0;
    }
    return pg;
  }
  __device__ __forceinline__ void at(int j, const T*& kr, const T*& vr) const {
    if constexpr (PAGED) {
      const int64_t pg = page_of(j), r = j & page_mask;
      kr = k + pg * k_sb + r * k_sn;
      vr = v + pg * v_sb + r * v_sn;
    } else {
      kr = k + j * k_sn;
      vr = v + j * v_sn;
    }
  }
};

template <typename T, bool PAGED>
__device__ __forceinline__ KeyRows<T, PAGED> key_rows(const DenseParams& p, int b, int kvh) {
  KeyRows<T, PAGED> r;
  const int64_t kb = PAGED ? 0 : b * p.k_sb, vb = PAGED ? 0 : b * p.v_sb;
  r.k = static_cast<const T*>(p.k) + kb + kvh * p.k_sh;
  r.v = static_cast<const T*>(p.v) + vb + kvh * p.v_sh;
  r.k_sn = p.k_sn;
  r.v_sn = p.v_sn;
  r.k_sb = p.k_sb;
  r.v_sb = p.v_sb;
  r.table = PAGED ? p.table + b * p.table_stride : nullptr;
  r.page_log2 = p.page_log2;
  r.page_mask = (1 << p.page_log2) - 1;
  r.num_pages = p.num_pages;
  r.error_flag = p.error_flag;
  return r;
}

// q . k over d elements in fp32 (rows of 16 bytes).
template <typename T>
__device__ __forceinline__ float row_dot(const T* a, const T* b, int d) {
  float s = 0.0f;
  for (int e = 0; e < d; e += 8) s = Op<T>::dot(Op<T>::load(a + e), Op<T>::load(b + e), s);
  return s;
}

template <typename T>
__device__ __forceinline__ float rule_of(const ScoreRule& r, float dot, float slope, int pos, int j) {
  float x = dot * r.c1;
  if (r.cap) x = r.c2 * cap_tanh<T>(x);
  return x - slope * fabsf(static_cast<float>(j - pos));
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

// Which (sequence, tile of rows) a block of a ragged batch takes: the idx-th
// tile in sequence order, sequences with at most few_rows rows left out.
// Returns false past the last one.
__device__ __forceinline__ bool find_tile(const DenseParams& p, int idx, int& b, int& tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int t = 0;
    if (b0 + lane < p.batch) {
      const int64_t rows = static_cast<int64_t>(paged_seq(p, b0 + lane).m) * p.g;
      t = rows > p.few_rows ? static_cast<int>((rows + kRows - 1) / kRows) : 0;
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

template <typename T, int D, bool PAGED, bool RULE>
__global__ __launch_bounds__(kThreads, 2) void dense_rows_kernel(DenseParams p) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int RB = D * O::kEsize;      // bytes of a tile row
  constexpr int NCH = RB / 16;           // its chunks
  constexpr int E = 16 / O::kEsize;      // elements of a chunk
  constexpr int KT = key_tile<T>();
  constexpr int NSUB = KT / 32, NC = D / 16, ND = D / 32;
  constexpr int RPP = kThreads / NCH;    // tile rows a pass of the block loads
  constexpr int NP = KT / RPP;
  constexpr int TB = KT * RB;            // bytes of a tile
  extern __shared__ __align__(16) char lds[];  // [2 buffers][K, V][TB]
  __shared__ int s_range[4][2];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int nbh = PAGED ? p.h_kv : p.batch * p.h_kv;
  const int w = blockIdx.x;
  const int bh = w % nbh;
  int rest = w / nbh;
  const int split = rest % p.splits;
  rest /= p.splits;
  int b, kvh, tile, first = 0, m;
  int64_t n_keys;
  if constexpr (PAGED) {
    kvh = bh;
    if (!find_tile(p, rest, b, tile)) return;
    const Seq s = paged_seq(p, b);
    first = s.first;
    m = s.m;
    n_keys = s.len;
    // the longest rows of a chunk first
    const int tiles = (m * p.g + kRows - 1) / kRows;
    tile = tiles - 1 - tile;
    if (tile < 0) return;
  } else {
    b = bh / p.h_kv;
    kvh = bh - b * p.h_kv;
    m = static_cast<int>(p.n_q);
    n_keys = p.n;
    const int tiles = static_cast<int>((p.n_q * p.g + kRows - 1) / kRows);
    tile = tiles - 1 - rest;
  }
  const KeyRows<T, PAGED> rows = key_rows<T, PAGED>(p, b, kvh);

  // this lane's row
  const int r = tile * kRows + wave * 32 + (lane & 31);
  const bool real = r < m * p.g;
  const int tok = real ? r / p.g : 0;
  const int hq = kvh * p.g + (real ? r - tok * p.g : 0);
  const int pos = PAGED ? static_cast<int>(n_keys) - m + tok : static_cast<int>(p.q_pos0) + tok;
  int lo = 0, hi = 0;
  if (real) {
    if (!PAGED && p.spans != nullptr) {
      const int2 s = p.spans[b * p.n_q + tok];
      lo = max(s.x, 0);
      hi = static_cast<int>(min(static_cast<int64_t>(s.y), n_keys));
    } else {
      hi = static_cast<int>(min(static_cast<int64_t>(pos) + 1, n_keys));
    }
    if (hi <= lo) lo = hi = 0;
  }
  const bool some = real && hi > lo;
  const float slope = (RULE && p.rule.slopes != nullptr && real) ? p.rule.slopes[hq] * kLog2e : 0.0f;
  const int lo_min = wave_min_i(some ? lo : 0x7FFFFFFF), hi_max = wave_max_i(some ? hi : 0);
  const int lo_max = wave_max_i(real ? lo : 0), hi_min = wave_min_i(real ? hi : 0x7FFFFFFF);
  if (lane == 0) {
    s_range[wave][0] = lo_min;
    s_range[wave][1] = hi_max;
  }
  __syncthreads();
  int k_lo = min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0]));
  int k_hi = max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1]));
  int part_lo = 0, part_hi = 0x7FFFFFFF;
  if (p.splits > 1) {
    const int64_t s0 = split * p.split_len, s1 = s0 + p.split_len;
    part_lo = static_cast<int>(min(s0, static_cast<int64_t>(0x7FFFFFFF)));
    part_hi = static_cast<int>(min(s1, static_cast<int64_t>(0x7FFFFFFF)));
    k_lo = max(k_lo, part_lo);
    k_hi = min(k_hi, part_hi);
  }
  const int t0 = k_lo / KT;
  const int nt = k_hi > k_lo ? (k_hi + KT - 1) / KT - t0 : 0;

  const T* qrow = static_cast<const T*>(p.q) + (PAGED ? first * p.q_sn : b * p.q_sb) + tok * p.q_sn + hq * p.q_sh;
  Frag qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = 16 * c + 8 * half;
    qf[c] = real && e < p.d ? O::load(qrow + e) : O::zero();
  }

  // staging: chunk sc of tile rows sr, sr + RPP, ...
  const int sc = tid % NCH, sr = tid / NCH;
  const bool chunk_ok = sc * E < p.d;
  uint4 kreg[NP], vreg[NP];
  auto load_tile = [&](int t) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int j = min((t0 + t) * KT + sr + i * RPP, static_cast<int>(n_keys) - 1);
      const T *kr, *vr;
      rows.at(j, kr, vr);
      kreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(kr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
      vreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(vr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto store_tile = [&](int buf) {
    char* kt = lds + buf * 2 * TB;
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

  if (nt > 0) {
    load_tile(0);
    store_tile(0);
  }
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) load_tile(t + 1);
    const int k0 = (t0 + t) * KT;
    if (k0 < hi_max && k0 + KT > lo_min) {
      const char* kt = lds + (t & 1) * 2 * TB;
      const char* vt = kt + TB;
      f32x16 s[NSUB];
#pragma unroll
      for (int u = 0; u < NSUB; ++u) s[u] = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < NSUB; ++u) s[u] = O::mfma(O::template row_frag<RB>(kt, 32 * u, c, lane), qf[c], s[u]);

      const int kl = k0 + 4 * half;  // key of register 0
      float cs = p.rule.c1;          // what is left to multiply the scores by
      if constexpr (RULE) {
        cs = 1.0f;
        if (p.rule.cap) {
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = p.rule.c2 * cap_tanh<T>(s[u][i] * p.rule.c1);
        } else {
#pragma unroll
          for (int u = 0; u < NSUB; ++u) s[u] *= p.rule.c1;
        }
        if (p.rule.slopes != nullptr) {
          const float dist = static_cast<float>(kl - pos);
#pragma unroll
          for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              s[u][i] = fmaf(-slope, fabsf(dist + static_cast<float>(32 * u + 8 * (i >> 2) + (i & 3))), s[u][i]);
        }
      }
      const bool whole = k0 >= lo_max && k0 + KT <= hi_min && k0 >= part_lo && k0 + KT <= part_hi;
      if (!whole) {
        const int a = max(lo, part_lo) - kl, z = min(hi, part_hi) - kl;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = 32 * u + 8 * (i >> 2) + (i & 3);
            if (j < a || j >= z) s[u][i] = -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
      top = fmaxf(top, other_half(top)) * cs;
      if (__ballot(top > mref + 8.0f) != 0) {
        const float mn = fmaxf(mref, top);
        const float alpha = mref == mn ? 1.0f : exp2_w(mref - mn);
        mref = mn;
        lsum *= alpha;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] *= alpha;
      }
      const float ref = mref == -INFINITY ? 0.0f : mref;
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[u][i] = exp2_w(fmaf(s[u][i], cs, -ref));
          lsum += s[u][i];
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
    if (t + 1 < nt) store_tile((t + 1) & 1);
  }

  // the row's sums, joined over the half-waves (they share the reference)
  lsum += other_half(lsum);
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) worst = finite(acc[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, other_half(worst));
  const bool again = some && (worst != 0.0f || !finite(lsum));
  const int64_t row_id = PAGED ? static_cast<int64_t>(first + tok) * p.h_q + hq
                               : (static_cast<int64_t>(b) * p.n_q + tok) * p.h_q + hq;
  // Where the row's result goes: the output, or its part.
  T* orow = static_cast<T*>(p.out) + (PAGED ? first * p.o_sn : b * p.o_sb) + tok * p.o_sn + hq * p.o_sh;
  T* low = p.out_low != nullptr ? static_cast<T*>(p.out_low) + (orow - static_cast<T*>(p.out)) : nullptr;
  float* prow = p.splits > 1 ? p.part_o + (split * p.part_rows + row_id) * D : nullptr;
  float* pml = p.splits > 1 ? p.part_ml + (split * p.part_rows + row_id) * 2 : nullptr;
  float* lrow = p.lse != nullptr ? p.lse + (static_cast<int64_t>(b) * p.h_q + hq) * p.n_q + tok : nullptr;

  // (a part whose visible keys all scored -inf says so by a finite m)
  const bool here = some && max(lo, part_lo) < min(hi, part_hi);
  if (real && !again) {
    if (p.splits > 1) {
      if (half == 0) {
        pml[0] = here && mref == -INFINITY ? -3.0e38f : mref;
        pml[1] = lsum;
      }
      if (lsum != 0.0f) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int dd = 32 * i + 8 * e + 4 * half;
            if (dd < p.d)
              *reinterpret_cast<float4*>(prow + dd) =
                  make_float4(acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]);
          }
      }
    } else {
      // no key: zeros; only keys of score -inf: NaN, as a softmax of them is
      const float inv = some ? 1.0f / lsum : 0.0f;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dd = 32 * i + 8 * e + 4 * half;
          if (dd < p.d) {
            const float a = acc[i][4 * e] * inv, c = acc[i][4 * e + 1] * inv, f = acc[i][4 * e + 2] * inv,
                        h = acc[i][4 * e + 3] * inv;
            O::store4(orow + dd, a, c, f, h);
            if (low != nullptr) O::store4(low + dd, O::left(a), O::left(c), O::left(f), O::left(h));
          }
        }
      if (lrow != nullptr && half == 0) *lrow = some ? mref + __log2f(lsum) : INFINITY;
    }
  }
  uint64_t todo = __ballot(again && half == 0);
  while (todo != 0) {  // rows to compute again, one after the other by the whole wave
    const int src = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int a = max(lane_value(lo, src), part_lo), z = min(lane_value(hi, src), part_hi);
    const int ps = lane_value(pos, src);
    const float sl = lane_value(slope, src);
    auto ptr_of = [&](const void* x) {
      const uint64_t u = reinterpret_cast<uint64_t>(x);
      return (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(u >> 32), src))) << 32) |
             static_cast<uint32_t>(lane_value(static_cast<int>(u & 0xFFFFFFFFu), src));
    };
    float o[4], mm, ll;
    exact_row<T, PAGED>(rows, p.rule, reinterpret_cast<const T*>(ptr_of(qrow)), p.d, a, z, sl, ps, o, mm, ll);
    const float inv = 1.0f / ll;
    if (p.splits > 1) {
      float* pr = reinterpret_cast<float*>(ptr_of(prow));
      float* pm = reinterpret_cast<float*>(ptr_of(pml));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < p.d) pr[lane + 64 * e] = o[e];
      if (lane == 0) {
        pm[0] = mm == -INFINITY ? -3.0e38f : mm;
        pm[1] = ll;
      }
    } else {
      T* orr = reinterpret_cast<T*>(ptr_of(orow));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < p.d) {
          O::store1(orr + lane + 64 * e, o[e] * inv);
          if (p.out_low != nullptr)
            O::store1(static_cast<T*>(p.out_low) + (orr - static_cast<T*>(p.out)) + lane + 64 * e, O::left(o[e] * inv));
        }
      float* lr = reinterpret_cast<float*>(ptr_of(lrow));
      if (lr != nullptr && lane == 0) *lr = mm + __log2f(ll);
    }
  }
}

// Joins the parts of each row: one wave a row, lane e features e, e + 64, ....
// A part without a key has m = -inf and l = 0 and its o is not read.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void dense_join_kernel(DenseParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.part_rows) return;
  float m = -INFINITY;
  bool seen = false;
  for (int s = lane; s < p.splits; s += 64) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * p.part_rows + row) * 2);
    if (ml.y != 0.0f) m = fmaxf(m, ml.x);
    seen |= ml.x != -INFINITY;
  }
  m = wave_max(m);
  seen = __ballot(seen) != 0;
  const float ref = m == -INFINITY ? 0.0f : m;
  float o[D / 64], l = 0.0f;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    float a = 0.0f, ls = 0.0f;
    if (s0 + lane < p.splits) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + ((s0 + lane) * p.part_rows + row) * 2);
      if (ml.y != 0.0f) {
        a = exp2_w(ml.x - ref);
        ls = ml.y * a;
      }
    }
    l += wave_sum(ls);
    uint64_t on = __ballot(ls != 0.0f);
    while (on != 0) {
      const int src = __builtin_ctzll(on);
      on &= on - 1;
      const float as = lane_value(a, src);
      const float* pr = p.part_o + ((s0 + src) * p.part_rows + row) * D;
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        if (lane + 64 * e < p.d) o[e] = fmaf(as, pr[lane + 64 * e], o[e]);
    }
  }
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
  T* orow = static_cast<T*>(p.out) + b * p.o_sb + t * p.o_sn + hq * p.o_sh;
  // no key: zeros; only keys of score -inf: NaN
  const float inv = seen ? 1.0f / l : 0.0f;
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    if (lane + 64 * e < p.d) {
      Op<T>::store1(orow + lane + 64 * e, o[e] * inv);
      if (p.out_low != nullptr)
        Op<T>::store1(static_cast<T*>(p.out_low) + (orow - static_cast<T*>(p.out)) + lane + 64 * e, Op<T>::left(o[e] * inv));
    }
  if (p.lse != nullptr && lane == 0) p.lse[(b * p.h_q + hq) * p.n_q + t] = seen ? m + __log2f(l) : INFINITY;
}

}  // namespace tile
}  // namespace ssa
