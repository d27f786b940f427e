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

// The row of key j: contiguous keys, or the sequence's pages (its new rows where the
// call brought them).
template <typename T, bool PAGED>
struct KeyRows {
  const T *k, *v;
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

template <typename T, bool PAGED>
__device__ __forceinline__ KeyRows<T, PAGED> key_rows(const DenseParams& p, int b, int kvh, int first, int cached) {
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

// FRESH: tiles of a paged call's own rows are read as contiguous ones are.
template <typename T, int D, bool PAGED, int RULE, int KW, bool FRESH = false>
__device__ __forceinline__ void dense_rows(const DenseParams& p, const int w, char* lds) {
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
  __shared__ int s_range[4][2];
  __shared__ float s_m[4][32], s_l[4][32];
  __shared__ int s_flag[4][32];

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
  const KeyRows<T, PAGED> rows = key_rows<T, PAGED>(p, b, kvh, first, static_cast<int>(n_keys) - m);

  // this lane's row
  const int r = tile * BR + rw * 32 + (lane & 31);
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
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const int lo_min = wave_min_i(some ? lo : 0x7FFFFFFF), hi_max = wave_max_i(some ? hi : 0);
  const int lo_max = wave_max_i(real ? lo : 0), hi_min = wave_min_i(real ? hi : 0x7FFFFFFF);
  if (lane == 0) {
    s_range[wave][0] = lo_min;
    s_range[wave][1] = hi_max;
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
  if (p.splits > 1) {
    const int64_t s0 = split * p.split_len, s1 = s0 + p.split_len;
    part_lo = static_cast<int>(min(s0, static_cast<int64_t>(0x7FFFFFFF)));
    part_hi = static_cast<int>(min(s1, static_cast<int64_t>(0x7FFFFFFF)));
    k_lo = max(k_lo, part_lo);
    k_hi = min(k_hi, part_hi);
  }
  const int t0 = k_lo / KT;
  const int nt = k_hi > k_lo ? (k_hi + KT - 1) / KT - t0 : 0;

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
  const int paged_end = PAGED ? min(rows.new_from, static_cast<int>(n_keys)) : 0;
  constexpr int RPW = 64 / NCH;  // rows of a wave's load
  auto find_pages = [&](int t) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < NP; ++i) pg[i] = rows.entry_of(min((t0 + t) * KT + i * RPP + wave * RPW, last));
    }
  };
  auto load_tile = [&](int t) {
    const int j0 = (t0 + t) * KT;
    if constexpr (PAGED) {
      if (j0 + KT <= paged_end) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int64_t page = rows.checked(__builtin_amdgcn_readfirstlane(pg[i])), r0 = (j0 + i * RPP + wave * RPW) & rows.page_mask;
          kreg[i] = row_load(row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes), koff);
          vreg[i] = row_load(row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes), voff);
        }
      } else if (FRESH && j0 >= rows.new_from) {
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
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const T *kr, *vr;
          rows.at(min(j0 + sr + i * RPP, last), kr, vr);
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
    find_pages(0);
    load_tile(0);
    if (nt > 1) find_pages(1);
    store_tile(0);
  }
  settle(qf);
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) load_tile(t + 1);
    if (t + 2 < nt) find_pages(t + 2);
    const int k0 = (t0 + t) * KT + kw * 32 * NSUB;
    if (k0 < hi_max && k0 + 32 * NSUB > lo_min) {
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
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[u][i] = rule.z(p.rule, s[u][i], slope, dist + static_cast<float>(32 * u + 8 * (i >> 2) + (i & 3)));
      const bool whole = k0 >= lo_max && k0 + 32 * NSUB <= hi_min && k0 >= part_lo && k0 + 32 * NSUB <= part_hi;
      if (!whole) {
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
    if (t + 1 < nt) store_tile(TWO ? (t + 1) & 1 : 0);
  }

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
  const bool here = some && max(lo, part_lo) < min(hi, part_hi);
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
    exact_row<T, PAGED>(rows, p.rule,
                        static_cast<const T*>(p.q) + (PAGED ? first * p.q_sn : b * p.q_sb) + tk * p.q_sn + h * p.q_sh, p.d, a,
                        z, sl, ps, o, mm, ll);
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
    if (lane == 0) put_sums(tk, h, mm, ll, true, a < z);
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
