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

#include <math.h>

#include "ssa_cuts.h"
#include "ssa_dense_rows.h"
#include "ssa_internal.h"

namespace ssa {
namespace {

using namespace tile;

constexpr int kAppend = 4 * kThreads;  // 16-byte chunks of a block that appends

// The sequence that holds a token: the last one that starts at or before it (-1 or batch: none).
__device__ __forceinline__ int sequence_of(const DenseParams& p, int tok) {
  int x = 0, y = p.batch + 1;  // the first start past the token
  while (x < y) {
    const int mid = (x + y) >> 1;
    if (p.starts[mid] <= tok)
      x = mid + 1;
    else
      y = mid;
  }
  return x - 1;
}

// One chunk of the new rows: k's first, then v's.
template <typename T>
__device__ __forceinline__ void append_chunk(const DenseParams& p, int64_t t) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int per = p.d / E;  // chunks of a row
  const int64_t total = p.n_q * p.h_kv * per;
  if (t >= 2 * total) return;
  const bool isv = t >= total;
  const int64_t u = isv ? t - total : t, row = u / per;
  const int c = static_cast<int>(u - row * per);
  const int tok = static_cast<int>(row / p.h_kv), h = static_cast<int>(row - static_cast<int64_t>(tok) * p.h_kv);
  const int b = sequence_of(p, tok);
  if (b < 0 || b >= p.batch) return;
  const Seq s = paged_seq(p, b);
  if (tok < s.first || tok >= s.first + s.m) return;
  const int j = s.len - s.m + tok - s.first;
  const int pg = p.table[b * p.table_stride + (j >> p.page_log2)];
  if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.num_pages)) {
    if (p.error_flag != nullptr) atomicOr(p.error_flag, 1);
    return;
  }
  const int64_t r = j & ((1 << p.page_log2) - 1);
  const T* src = static_cast<const T*>(isv ? p.v_new : p.k_new) + tok * (isv ? p.vn_st : p.kn_st) +
                 h * (isv ? p.vn_sh : p.kn_sh) + c * E;
  T* dst = static_cast<T*>(const_cast<void*>(isv ? p.v : p.k)) + pg * (isv ? p.v_sb : p.k_sb) +
           r * (isv ? p.v_sn : p.k_sn) + h * (isv ? p.v_sh : p.k_sh) + c * E;
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
}

// Zeros to the rows of out of a block's tokens, one a thread, that no sequence has, or one
// that is left out.
template <typename T>
__device__ __forceinline__ void no_rows(const DenseParams& p, const int block) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 63, per = p.d / E;
  const int64_t tok0 = static_cast<int64_t>(block) * blockDim.x + (threadIdx.x & ~63);
  bool none = false;
  if (tok0 + lane < p.n_q) {
    const int tok = static_cast<int>(tok0) + lane, b = sequence_of(p, tok);
    none = true;
    if (b >= 0 && b < p.batch) {
      const Seq s = paged_seq(p, b);
      none = tok < s.first || tok >= s.first + s.m;
    }
  }
  for (uint64_t todo = __ballot(none); todo != 0; todo &= todo - 1) {
    T* row = static_cast<T*>(p.out) + (tok0 + __builtin_ctzll(todo)) * p.o_sn;
    for (int c = lane; c < p.h_q * per; c += 64) {
      const int h = c / per;
      *reinterpret_cast<uint4*>(row + h * p.o_sh + (c - h * per) * E) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

template <typename T, int D, int RULE>
__device__ __forceinline__ void few_rows(const DenseParams& p, const int block, char* lds) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int RB = D * O::kEsize, NCH = RB / 16, E = 16 / O::kEsize;
  constexpr int NC = D / 16, ND = D / 32, TB = 32 * RB;
  constexpr int RPW = 64 / NCH, NP = 32 / RPW;  // rows a wave's load instruction covers; loads of a tile
  constexpr int PS = D + 4;                     // floats of a row of partial sums
  // lds: [4 waves][K, V][TB], then [4][32][PS] sums
  __shared__ float s_m[4][kFew], s_l[4][kFew];
  __shared__ int s_bad[4][kFew];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = block % p.h_kv;
  const int rest = block / p.h_kv;
  const int split = rest % p.splits, b = rest / p.splits;
  const Seq sq = paged_seq(p, b);
  const int R = sq.m * p.g;
  if (R == 0 || R > p.few_rows) return;
  const int k_begin = static_cast<int>(min(split * p.split_len, static_cast<int64_t>(sq.len)));
  const int k_end = static_cast<int>(min((split + 1) * p.split_len, static_cast<int64_t>(sq.len)));
  if (k_begin >= k_end) return;  // (a part past the sequence, which the join does not read)
  const KeyRows<T, true> rows = key_rows<T, true>(p, b, kvh, sq.first, sq.len - sq.m);

  const int rr = lane & 31;
  const bool real = rr < R;
  const int tok = real ? rr / p.g : 0;
  const int hq = kvh * p.g + (real ? rr - tok * p.g : 0);
  const int pos = sq.len - sq.m + tok;
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const T* qrow = static_cast<const T*>(p.q) + (sq.first + tok) * p.q_sn + hq * p.q_sh;
  Frag qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = 16 * c + 8 * half;
    qf[c] = real && e < p.d ? O::load(qrow + e) : O::zero();
  }

  char* kt = lds + wave * 2 * TB;
  char* vt = kt + TB;
  const int sc = lane % NCH, sr = lane / NCH;
  const bool chunk_ok = sc * E < p.d;
  uint4 kreg[NP], vreg[NP];
  auto pages_at = [&](int k0) { return k0 < k_end ? rows.entry_of(min(k0 + rr, k_end - 1)) : 0; };
  auto load_tile = [&](int k0, int entry) {
    const int pg = rows.checked(entry);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = sr + i * RPW;
      const T *kr, *vr;
      rows.in_page(__shfl(pg, r, 64), min(k0 + r, k_end - 1), kr, vr);
      kreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(kr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
      vreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(vr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
    }
  };

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{};
  float mref = -INFINITY, lsum = 0.0f;

  int k0 = k_begin + 32 * wave;
  int pg = pages_at(k0);
  if (k0 < k_end) load_tile(k0, pg);
  pg = pages_at(k0 + 128);
  settle(qf);
  for (; k0 < k_end; k0 += 128) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = chunk_at<RB>(sr + i * RPW, sc);
      *reinterpret_cast<uint4*>(kt + at) = kreg[i];
      *reinterpret_cast<uint4*>(vt + at) = vreg[i];
    }
    wave_lds_sync();
    if (k0 + 128 < k_end) load_tile(k0 + 128, pg);
    pg = pages_at(k0 + 256);
    f32x16 s = f32x16{};
#pragma unroll
    for (int c = 0; c < NC; ++c) s = O::mfma(O::template row_frag<RB>(kt, 0, c, lane), qf[c], s);
    const int kl = k0 + 4 * half;
    const float dist = static_cast<float>(kl - pos);
    const int z = min(pos + 1, k_end) - kl;
    float top = Rule<T, RULE>::kHidden;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = 8 * (i >> 2) + (i & 3);
      s[i] = rule.z(p.rule, s[i], slope, dist + static_cast<float>(j));
      if (j >= z) s[i] = Rule<T, RULE>::kHidden;
      top = rule.better(top, s[i]);
    }
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
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_w(fmaf(s[i], rule.a, nref));
      lsum += s[i];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Frag pf = O::pack(s, c);
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[i] = O::mfma(O::template col_frag<RB>(vt, 16 * c, 32 * i, lane), pf, acc[i]);
    }
    wave_lds_sync();
  }

  lsum += other_half(lsum);
  float worst = finite(lsum) ? 0.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) worst = finite(acc[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, other_half(worst));
  if (half == 0) {
    s_m[wave][rr] = mref;
    s_l[wave][rr] = lsum;
    s_bad[wave][rr] = worst != 0.0f;
  }
  __syncthreads();  // every wave is past its tiles: their LDS holds the sums now
  float* sums = reinterpret_cast<float*>(lds);
  if (real) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(sums + (wave * kFew + rr) * PS + 32 * i + 8 * e + 4 * half) =
            make_float4(acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]);
  }
  __syncthreads();
  const int64_t part_row = (static_cast<int64_t>(b) * p.h_kv + kvh) * kFew;
  const int quads = p.d / 4;
  for (int e = tid; e < R * quads; e += kThreads) {
    const int r = e / quads, dd = (e - r * quads) * 4;
    if (s_bad[0][r] | s_bad[1][r] | s_bad[2][r] | s_bad[3][r]) continue;
    const float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float ref = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float a = exp2_w(s_m[x][r] - ref);
      const float4 t = *reinterpret_cast<const float4*>(sums + (x * kFew + r) * PS + dd);
      l = fmaf(a, s_l[x][r], l);
      o.x = fmaf(a, t.x, o.x);
      o.y = fmaf(a, t.y, o.y);
      o.z = fmaf(a, t.z, o.z);
      o.w = fmaf(a, t.w, o.w);
    }
    const int t = r / p.g, h = kvh * p.g + r - t * p.g;
    if (p.splits > 1) {
      const int64_t pr = split * p.part_rows + part_row + r;
      *reinterpret_cast<float4*>(p.part_o + pr * D + dd) = o;
      if (dd == 0) {
        // (a part whose visible keys all scored -inf says so by a finite m)
        const bool here = k_begin < min(k_end, sq.len - sq.m + t + 1);
        p.part_ml[pr * 2] = here && m == -INFINITY ? -3.0e38f : m;
        p.part_ml[pr * 2 + 1] = l;
      }
    } else {
      const float inv = 1.0f / l;
      T* orow = static_cast<T*>(p.out) + (sq.first + t) * p.o_sn + h * p.o_sh;
      O::store4(orow + dd, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
  }
  for (int r = wave; r < R; r += 4) {  // rows to compute again, key by key
    if (!(s_bad[0][r] | s_bad[1][r] | s_bad[2][r] | s_bad[3][r])) continue;
    const int t = r / p.g, h = kvh * p.g + r - t * p.g, ps = sq.len - sq.m + t;
    const float sl = has_bias(RULE) ? slope_of(p.rule, h) : 0.0f;
    float o[4], m, l;
    exact_row<T, true>(rows, p.rule, static_cast<const T*>(p.q) + (sq.first + t) * p.q_sn + h * p.q_sh, p.d, k_begin,
                       min(k_end, ps + 1), sl, ps, o, m, l);
    const int64_t pr = split * p.part_rows + part_row + r;
    T* orow = static_cast<T*>(p.out) + (sq.first + t) * p.o_sn + h * p.o_sh;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const int dd = lane + 64 * e;
      if (dd >= p.d) continue;
      if (p.splits > 1)
        p.part_o[pr * D + dd] = o[e];
      else
        O::store1(orow + dd, o[e] * (1.0f / l));
    }
    if (p.splits > 1 && lane == 0) {
      p.part_ml[pr * 2] = k_begin < min(k_end, ps + 1) && m == -INFINITY ? -3.0e38f : m;
      p.part_ml[pr * 2 + 1] = l;
    }
  }
}

// Everything of a call in one launch: blocks of many rows (the longest) first, then
// few rows, then the blocks that append.  KW 0: no sequence has many rows; its call may
// have no second launch, so that the blocks of no rows stand here (beside dense_rows they
// cost 2048 rows behind 30720 cached 12%: 1215 to 1350 us).
template <typename T, int D, int KW>
constexpr int paged_per_cu() {
  if constexpr (KW > 0) return rows_per_cu<T, D, KW>();
  return sizeof(T) == 2 || D == 64 ? 2 : 1;
}

template <typename T, int D, int RULE, int KW, bool FRESH>
__global__ __launch_bounds__(kThreads, (paged_per_cu<T, D, KW>())) void paged_kernel(DenseParams rows, DenseParams few, int row_blocks,
                                                                                     int few_blocks, int copy_blocks) {
  extern __shared__ __align__(16) char lds[];
  const int w = blockIdx.x;
  if (w < row_blocks) {
    if constexpr (KW > 0) dense_rows<T, D, true, RULE, KW, FRESH>(rows, w, lds);
  } else if (w < row_blocks + few_blocks) {
    few_rows<T, D, RULE>(few, w - row_blocks, lds);
  } else if (KW > 0 || w < row_blocks + few_blocks + copy_blocks) {
    const int64_t t = static_cast<int64_t>(w - row_blocks - few_blocks) * kAppend + threadIdx.x;
    for (int i = 0; i < kAppend; i += kThreads) append_chunk<T>(few, t + i);
  } else {
    if constexpr (KW == 0) no_rows<T>(few, w - row_blocks - few_blocks - copy_blocks);
  }
}

// The parts of few-row sequences: `per` waves a row (1, 4 or 16 of the block's 16),
// each with every per-th part, eight parts' loads in flight; their sums meet in LDS.
constexpr int kJoinWaves = 16, kAtOnce = 8;

template <typename T, int D>
__device__ __forceinline__ void few_join(const DenseParams& p, const int block, const int most_rows, const int per) {
  constexpr int L = D / 64;  // features of a lane: lane * L ..
  __shared__ float s_o[kJoinWaves][D], s_m[kJoinWaves], s_l[kJoinWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t x = static_cast<int64_t>(block) * (kJoinWaves / per) + wave / per;
  const int bh = static_cast<int>(x / most_rows), r = static_cast<int>(x - static_cast<int64_t>(bh) * most_rows);
  const int b = min(bh / p.h_kv, p.batch - 1), kvh = bh - b * p.h_kv;
  const Seq sq = paged_seq(p, b);
  const int R = sq.m * p.g;
  const bool on = bh < p.batch * p.h_kv && R <= p.few_rows && r < R;
  const int parts = on ? static_cast<int>(min(static_cast<int64_t>(p.splits), ceil_div(sq.len, p.split_len))) : 0;
  const int64_t row = static_cast<int64_t>(bh) * kFew + r;
  float m = -INFINITY, l = 0.0f, o[L];
#pragma unroll
  for (int e = 0; e < L; ++e) o[e] = 0.0f;
  for (int s0 = wave % per; s0 < parts; s0 += kAtOnce * per) {
    float2 ml[kAtOnce];
    float v[kAtOnce][L];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = min(s0 + i * per, parts - 1) * p.part_rows + row;
      ml[i] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
#pragma unroll
      for (int e = 0; e < L; ++e) v[i][e] = p.part_o[at * D + lane * L + e];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (s0 + i * per >= parts || ml[i].y == 0.0f) continue;  // (an empty part)
      const float mn = fmaxf(m, ml[i].x), ref = mn == -INFINITY ? 0.0f : mn;
      const float a = exp2_w(m - ref), w = exp2_w(ml[i].x - ref);
      m = mn;
      l = fmaf(l, a, ml[i].y * w);
#pragma unroll
      for (int e = 0; e < L; ++e) o[e] = fmaf(v[i][e], w, o[e] * a);
    }
  }
  if (per > 1) {
#pragma unroll
    for (int e = 0; e < L; ++e) s_o[wave][lane * L + e] = o[e];
    if (lane == 0) {
      s_m[wave] = m;
      s_l[wave] = l;
    }
    __syncthreads();
    if (wave % per != 0) return;
    float top = m;
    for (int y = 1; y < per; ++y) top = fmaxf(top, s_m[wave + y]);
    const float ref = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < L; ++e) o[e] = 0.0f;
    for (int y = 0; y < per; ++y) {
      const float a = exp2_w(s_m[wave + y] - ref);
      l = fmaf(a, s_l[wave + y], l);
#pragma unroll
      for (int e = 0; e < L; ++e) o[e] = fmaf(a, s_o[wave + y][lane * L + e], o[e]);
    }
  }
  if (!on) return;
  const int t = r / p.g, h = kvh * p.g + r - t * p.g;
  T* orow = static_cast<T*>(p.out) + (sq.first + t) * p.o_sn + h * p.o_sh;
  const float inv = 1.0f / l;  // (a token sees itself: the sum is 0 only where every score is -inf)
#pragma unroll
  for (int e = 0; e < L; ++e)
    if (lane * L + e < p.d) Op<T>::store1(orow + lane * L + e, o[e] * inv);
}

// The parts of both kinds of rows, in one launch, and the rows without a sequence.
template <typename T, int D>
__global__ __launch_bounds__(kJoinWaves * 64) void paged_join_kernel(DenseParams rows, DenseParams few, int few_blocks,
                                                                          int join_blocks, int most_rows, int per) {
  if (static_cast<int>(blockIdx.x) < few_blocks)
    few_join<T, D>(few, blockIdx.x, most_rows, per);
  else if (static_cast<int>(blockIdx.x) >= join_blocks)
    no_rows<T>(few, blockIdx.x - join_blocks);
  else
    dense_join<T, D>(rows, static_cast<int64_t>(blockIdx.x - few_blocks) * kJoinWaves + (threadIdx.x >> 6));
}

template <typename T, int D, int RULE, int KW, bool FRESH = false>
int launch_paged(DenseParams& p, const PagedPlan& l, bool zero_rows, char* ws, hipStream_t st) {
  const char* fn = "ssa_paged_step";
  DenseParams f = p, r = p;
  f.splits = l.few_splits;
  f.split_len = l.few_len;
  f.part_rows = static_cast<int64_t>(p.batch) * p.h_kv * kFew;
  f.part_o = reinterpret_cast<float*>(ws + l.few_o);
  f.part_ml = reinterpret_cast<float*>(ws + l.few_ml);
  r.splits = l.row_splits;
  r.split_len = l.row_len;
  r.part_rows = p.n_q * p.h_q;
  r.part_o = reinterpret_cast<float*>(ws + l.row_o);
  r.part_ml = reinterpret_cast<float*>(ws + l.row_ml);
  const size_t tiles = static_cast<size_t>(8) * 32 * D * sizeof(T), sums = static_cast<size_t>(4) * kFew * (D + 4) * sizeof(float);
  size_t bytes = tiles > sums ? tiles : sums;
  if constexpr (KW > 0) bytes = bytes > rows_lds<T, D, KW>() ? bytes : rows_lds<T, D, KW>();
  if (int rc = reserve_lds(reinterpret_cast<const void*>(paged_kernel<T, D, RULE, KW, FRESH>), bytes + 4096, fn)) return rc;
  const int64_t rblocks = static_cast<int64_t>(l.row_tiles) * p.h_kv * r.splits;
  const int64_t fblocks = static_cast<int64_t>(p.batch) * p.h_kv * f.splits;
  const int64_t chunks = p.k_new == nullptr ? 0 : 2 * p.n_q * p.h_kv * (p.d / (16 / static_cast<int>(sizeof(T))));
  const int most = static_cast<int>(p.max_new * p.g < kFew ? p.max_new * p.g : kFew);
  const int per = f.splits <= 8 ? 1 : (f.splits <= 32 ? 4 : 16);  // waves a row: one round of loads, or 16 waves
  const int64_t few_join_blocks = f.splits > 1 ? ceil_div(static_cast<int64_t>(p.batch) * p.h_kv * most, kJoinWaves / per) : 0;
  const int64_t join_blocks = few_join_blocks + (l.row_tiles > 0 && r.splits > 1 ? ceil_div(r.part_rows, kJoinWaves) : 0);
  const bool zero_here = zero_rows && KW == 0 && join_blocks == 0;
  const int64_t second = join_blocks + (zero_rows && !zero_here ? ceil_div(p.n_q, kJoinWaves * 64) : 0);
  if (second > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many sequences", fn);
  const int64_t cblocks = ceil_div(chunks, kAppend);
  const int64_t blocks = rblocks + fblocks + cblocks + (zero_here ? ceil_div(p.n_q, kThreads) : 0);
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  paged_kernel<T, D, RULE, KW, FRESH><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), bytes, st>>>(
      r, f, static_cast<int>(rblocks), static_cast<int>(fblocks), static_cast<int>(cblocks));
  if (int rc = check_launch("ssa_paged_step")) return rc;
  if (second > 0) {
    paged_join_kernel<T, D><<<dim3(static_cast<unsigned>(second)), dim3(kJoinWaves * 64), 0, st>>>(
        r, f, static_cast<int>(few_join_blocks), static_cast<int>(join_blocks), most, per);
    return check_launch("ssa_paged_step join");
  }
  return SSA_OK;
}

template <typename T, int D, int RULE>
int launch_kw(DenseParams& p, const PagedPlan& l, bool zero, char* ws, hipStream_t st) {
  if (l.row_tiles == 0) return launch_paged<T, D, RULE, 0>(p, l, zero, ws, st);
  // Where a good part of the keys are the call's own rows, their tiles are read as
  // contiguous ones (four prompts of 1000 tokens, 32 / 8 heads: 117 to 81 us); the
  // branch costs the pages' tiles 16% (2048 tokens behind 30720: 1220 to 1410).
  const bool fresh = p.k_new != nullptr && 3 * p.max_new >= p.max_len;
  if constexpr (most_kw<T, D>() >= 4)
    if (l.row_kw == 4) return fresh ? launch_paged<T, D, RULE, 4, true>(p, l, zero, ws, st) : launch_paged<T, D, RULE, 4>(p, l, zero, ws, st);
  if (l.row_kw == 2) return fresh ? launch_paged<T, D, RULE, 2, true>(p, l, zero, ws, st) : launch_paged<T, D, RULE, 2>(p, l, zero, ws, st);
  return fresh ? launch_paged<T, D, RULE, 1, true>(p, l, zero, ws, st) : launch_paged<T, D, RULE, 1>(p, l, zero, ws, st);
}

template <typename T, int D>
int launch_rule(DenseParams& p, const PagedPlan& l, bool zero, char* ws, hipStream_t st) {
  switch (rule_kind<T>(p.rule)) {
    case kPlain: return launch_kw<T, D, kPlain>(p, l, zero, ws, st);
    case kCap: return launch_kw<T, D, kCap>(p, l, zero, ws, st);
    case kBias: return launch_kw<T, D, kBias>(p, l, zero, ws, st);
    case kFar:
      if constexpr (sizeof(T) == 2) return launch_kw<T, D, kFar>(p, l, zero, ws, st);
  }
  return fail(SSA_ERR_UNSUPPORTED, "no kernel for this rule of scores");
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" size_t ssa_paged_step_workspace_bytes(int dtype, int64_t tokens, int64_t batch, int h_q, int h_kv, int d,
                                                 int64_t max_new, int64_t max_len) {
  if (tokens <= 0 || batch <= 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0 || max_new <= 0 || max_len <= 0) return 0;
  // (what the call refuses: products of these would overflow, to a division by zero at worst)
  if (tokens > 0x7FFFFF00 || batch > 0x7FFFFF || max_len > 0x7FFFFF00) return 0;
  return paged_plan(dtype, tokens, batch, h_q, h_kv, d, max_new, max_len).bytes;
}

static int paged_step(const char* fn, bool zero_rows, const void* q, const void* k, const void* v, int dtype,
                      int64_t tokens, int64_t batch, int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st,
                      int64_t k_sh, int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages,
                      int page_size, int64_t kp_sp, int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st,
                      int64_t vp_sh, const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                      const int32_t* cached, int64_t max_new, int64_t max_len, float scale_div, float softcap,
                      const float* slopes, void* out, int64_t o_st, int64_t o_sh, int32_t* error_flag, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (int rc = check_heads(fn, dtype, h_q, h_kv, d)) return rc;
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
  if (int rc = check_aligned(fn, "k_pages", dtype, k_pages, kp_sp, kp_st, kp_sh)) return rc;
  if (int rc = check_aligned(fn, "v_pages", dtype, v_pages, vp_sp, vp_st, vp_sh)) return rc;
  if (int rc = check_aligned(fn, "out", dtype, out, 0, o_st, o_sh)) return rc;
  const PagedPlan l = paged_plan(dtype, tokens, batch, h_q, h_kv, d, max_new, max_len);
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
  p.max_new = max_new < tokens ? max_new : tokens; p.max_len = max_len;
  p.error_flag = error_flag;
  p.k_new = k; p.v_new = v;
  p.kn_st = k_st; p.kn_sh = k_sh; p.vn_st = v_st; p.vn_sh = v_sh;
  hipStream_t st = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  if (dtype == SSA_DTYPE_F32)
    return d <= 64 ? launch_rule<float, 64>(p, l, zero_rows, ws, st) : launch_rule<float, 128>(p, l, zero_rows, ws, st);
  return d <= 64 ? launch_rule<uint16_t, 64>(p, l, zero_rows, ws, st) : launch_rule<uint16_t, 128>(p, l, zero_rows, ws, st);
}

extern "C" int ssa_paged_step(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch,
                              int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                              int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages, int page_size,
                              int64_t kp_sp, int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh,
                              const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                              const int32_t* cached, int64_t max_new, int64_t max_len, float scale_div, float softcap,
                              const float* slopes, void* out, int64_t o_st, int64_t o_sh, int32_t* error_flag,
                              void* workspace, size_t workspace_bytes, void* stream) {
  return paged_step("ssa_paged_step", false, q, k, v, dtype, tokens, batch, h_q, h_kv, d, q_st, q_sh, k_st, k_sh, v_st,
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
  return paged_step("ssa_paged_step_zeroed", true, q, k, v, dtype, tokens, batch, h_q, h_kv, d, q_st, q_sh, k_st, k_sh,
                    v_st, v_sh, k_pages, v_pages, num_pages, page_size, kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh, table,
                    table_stride, max_pages, starts, cached, max_new, max_len, scale_div, softcap, slopes, out, o_st, o_sh,
                    error_flag, workspace, workspace_bytes, stream);
}
