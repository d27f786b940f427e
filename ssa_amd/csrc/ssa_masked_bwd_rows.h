// Gradients of dense attention with a key interval per row
// (ssa_masked_attention_backward).  With s the score rule's scores, t the cap's
// tanh (0 without), p = exp(s - lse) over the visible keys, D_i = dO_i . o_i:
//
//   dV_j = sum_i p_ij dO_i          dS_ij = p_ij (dO_i . v_j - D_i) (1 - t_ij^2)
//   dQ_i = sum_j dS_ij k_j / scale  dK_j  = sum_i dS_ij q_i / scale
//
// D takes a bf16 output with what its rounding left (out_low): from the rounded
// one alone, D's error enters every dS of the row, and with few keys a row dq and
// dk end 1.7 times as far from 64 bits as their own rounding puts them (1.45 with
// it; 2^-8 roundings of P and dS are the rest).
//
// Two kernels and no atomics, so the sums' order is fixed: dq_kernel by rows
// (S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T), which also writes D and each
// 32-row group's interval bounds, then dkv_kernel by keys (S = Q K^T, dP = dO
// V^T, dV^T += dO^T P, dK^T += Q^T dS) over the rows of all g query heads, so a
// shared head's gradient is summed in its block.  S and dP are computed twice:
// 7 products for the 5 of a single kernel, whose dQ would need fp32 atomics
// (read-modify-writes of n x h_q x d floats for every 128 keys, and sums whose
// order changes from run to run).
//
// Bound by the matrix cores and the vector unit's exponentials beside them (32 / 8
// heads, bf16, of the 7 products that it does; a library product: 1.13 PFLOP/s):
//   8192 x 8192, d = 128              3.8 ms, 1.02 PFLOP/s; d = 64 2.14 ms, 0.90
//   4096 x 4096, 16 / 4 heads, fp32   1.87 ms (d = 64), 129 of the product's 154 TFLOP/s
// and on packed documents by blocks of unlike lengths: twelve in 8192 tokens 0.22 ms
// (dQ) and 0.44 ms (dK, dV), 0.43 PFLOP/s.
//
// Of bf16 calls P and dS are rounded to bf16 (half a step, 2^-8 of each) for the products that make dV, dQ
// and dK, whose sums are fp32; scores, dO . V and D are fp32.
//
// Rows that see two intervals (kTwo: a sliding window and a document's first keys): dQ walks
// the tiles of both.  For dK and dV the first keys of a document are seen by all of its rows
// and others by a window of them, 14 times as few where 16384 rows see 1024 keys back, so that
// blocks of equal keys are not blocks of equal work.  Two small kernels look at the groups'
// bounds first: plan_count counts the row tiles that see each block of keys, plan_list cuts blocks
// with more than their share of all of them into parts (and gives these slots of the workspace).
// Only cut blocks of keys go through fp32 parts.
//
// Masked rows or keys that hold infinities or NaN: as in the forward, sums that
// end up other than finite are computed again pair by pair, visible pairs only.
#pragma once

#include <math.h>

#include "ssa_cuts.h"
#include "ssa_dense_rows.h"
#include "ssa_internal.h"

namespace ssa {
namespace {

using namespace tile;

struct BwdParams {
  const void *q, *k, *v, *out, *out_low, *dout;
  const float* lse;
  void *dq, *dk, *dv;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, o_sb, o_sn, o_sh, do_sb, do_sn, do_sh;
  int64_t n, n_q, q_pos0;
  int batch, h_q, h_kv, g, d;
  const int2* spans;
  ScoreRule rule;
  float inv_scale;
  float4* stats;  // [batch][h_q][n_q]: lse, D, lo, hi (the last two as ints)
  int4* bounds;   // [batch][groups of 32 packed rows]: lo_min, hi_max, lo_max, hi_min
  int groups;
  int splits;     // parts of the rows for dK and dV
  float *part_k, *part_v;  // [splits][batch][n][h_kv][D]
  // kTwo (spans hold two intervals a row, bounds two records a group): blocks of keys of all
  // batch elements, how many tiles of rows see each, and what the blocks of dkv_kernel take
  int key_blocks, key_tiles, extra;
  int* counts;      // [key_blocks]: row tiles that see it
  int4* entries;    // [key_blocks + most]: block of keys (-1: nothing), part, parts, first slot
  int4* cut;        // how many, then of each its block of keys (-1: in one part), parts, first slot
};

constexpr int kBlk = 128;  // rows or keys of a block

__device__ __forceinline__ int2 row_span(const BwdParams& p, int b, int tok) {
  int lo = 0, hi;
  if (p.spans != nullptr) {
    const int2 s = p.spans[b * p.n_q + tok];
    lo = max(s.x, 0);
    hi = static_cast<int>(min(static_cast<int64_t>(s.y), p.n));
  } else {
    hi = static_cast<int>(min(p.q_pos0 + tok + 1, p.n));
  }
  return hi > lo ? make_int2(lo, hi) : make_int2(0, 0);
}

// kTwo: the row's second interval [x, y) and another [z, w), both clamped; one interval alone is
// the first.
__device__ __forceinline__ int4 row_sets(const BwdParams& p, int b, int tok) {
  const int4 s = reinterpret_cast<const int4*>(p.spans)[b * p.n_q + tok];
  int lo = max(s.x, 0), hi = static_cast<int>(min(static_cast<int64_t>(s.y), p.n));
  int x = max(s.z, 0), y = static_cast<int>(min(static_cast<int64_t>(s.w), p.n));
  if (hi <= lo) lo = hi = 0;
  if (y <= x) x = y = 0;
  return hi > lo ? make_int4(lo, hi, x, y) : make_int4(x, y, 0, 0);
}

// x (log2 units) and 1 - t^2 of a raw product, one pair at a time.
template <typename T>
__device__ __forceinline__ float score_x(const ScoreRule& r, float dot, float slope, float dist, float& factor) {
  if (sizeof(T) == 2 && r.cap == kSeries) return Rule<T, kFar>(r).z(r, dot, slope, dist, factor);
  return Rule<T, kBias>(r).z(r, dot, slope, dist, factor);
}

__device__ __forceinline__ const void* lane_ptr(const void* x, int src) {
  const uint64_t u = reinterpret_cast<uint64_t>(x);
  return reinterpret_cast<const void*>(
      (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(u >> 32), src))) << 32) |
      static_cast<uint32_t>(lane_value(static_cast<int>(u & 0xFFFFFFFFu), src)));
}

template <typename T, int D, int KW>
constexpr int dq_keys() {
  return KW > 1 ? 32 * KW : (sizeof(T) == 2 ? 64 : 32);
}
// LDS: two buffers of K and V, or at the end the sums of the waves that share rows.
template <typename T, int D, int KW>
constexpr size_t dq_lds() {
  const size_t tiles = static_cast<size_t>(4) * dq_keys<T, D, KW>() * D * sizeof(T);
  const size_t sums = KW > 1 ? static_cast<size_t>(4) * 32 * (D + 4) * sizeof(float) : 0;
  return tiles > sums ? tiles : sums;
}

template <typename T, int D, int RULE, int KW, int VIEW>
__global__ __launch_bounds__(kThreads, (dq_lds<T, D, KW>() > 80 * 1024 || (sizeof(T) == 4 && D == 128) ? 1 : 2)) void dq_kernel(BwdParams p) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr bool SETS = VIEW == kTwo;
  constexpr int RB = D * O::kEsize, NCH = RB / 16, E = 16 / O::kEsize;
  constexpr int KT = dq_keys<T, D, KW>();
  constexpr int NSUB = KT / (32 * KW), NC = D / 16, ND = D / 32, BR = kBlk / KW, PS = D + 4;
  constexpr int RPP = kThreads / NCH, NP = KT / RPP, TB = KT * RB;
  extern __shared__ __align__(16) char lds[];
  __shared__ int s_range[4][SETS ? 4 : 2];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave % KW, rw = wave / KW;
  const int nbh = p.batch * p.h_kv;
  const int bh = blockIdx.x % nbh;
  const int tiles = static_cast<int>((p.n_q * p.g + BR - 1) / BR);
  const int tile = tiles - 1 - static_cast<int>(blockIdx.x / nbh);
  const int b = bh / p.h_kv, kvh = bh - b * p.h_kv;
  const int n_keys = static_cast<int>(p.n);

  const int r = tile * BR + rw * 32 + (lane & 31);
  const bool real = r < p.n_q * p.g;
  const int tok = real ? r / p.g : 0;
  const int hq = kvh * p.g + (real ? r - tok * p.g : 0);
  const int pos = static_cast<int>(p.q_pos0) + tok;
  int4 sp = make_int4(0, 0, 0, 0);
  if (real) {
    if constexpr (SETS) {
      sp = row_sets(p, b, tok);
    } else {
      const int2 one = row_span(p, b, tok);
      sp.x = one.x;
      sp.y = one.y;
    }
  }
  const int lo = sp.x, hi = sp.y;
  const bool some = real && hi > lo;
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const int lo_min = wave_min_i(some ? lo : 0x7FFFFFFF), hi_max = wave_max_i(some ? hi : 0);
  const int lo_max = wave_max_i(real ? lo : 0), hi_min = wave_min_i(real ? hi : 0x7FFFFFFF);
  int a_min = 0x7FFFFFFF, a_max = 0;
  if constexpr (SETS) {
    a_min = wave_min_i(sp.w > sp.z ? sp.z : 0x7FFFFFFF);
    a_max = wave_max_i(sp.w);
  }
  if (lane == 0) {
    s_range[wave][0] = lo_min;
    s_range[wave][1] = hi_max;
    if constexpr (SETS) {
      s_range[wave][2] = a_min;
      s_range[wave][3] = a_max;
    }
    const int grp = tile * (BR / 32) + rw;
    if (kvh == 0 && kw == 0 && grp < p.groups) {
      int4* to = p.bounds + (static_cast<int64_t>(b) * p.groups + grp) * (SETS ? 2 : 1);
      to[0] = make_int4(lo_min, hi_max, lo_max, hi_min);
      if constexpr (SETS) to[1] = make_int4(a_min, a_max, 0, 0);
    }
  }
  __syncthreads();
  const int k_lo = __builtin_amdgcn_readfirstlane(min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0])));
  const int k_hi = __builtin_amdgcn_readfirstlane(max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1])));
  Tiles walk{k_lo / KT, 0, 0, 0};
  if constexpr (SETS) {
    const int x = __builtin_amdgcn_readfirstlane(min(min(s_range[0][2], s_range[1][2]), min(s_range[2][2], s_range[3][2])));
    const int y = __builtin_amdgcn_readfirstlane(max(max(s_range[0][3], s_range[1][3]), max(s_range[2][3], s_range[3][3])));
    const int z = k_hi > k_lo ? k_lo : 0;
    walk = y > x ? tiles_of(x, y, z, k_hi, KT) : tiles_of(0, 0, z, k_hi, KT);
  }
  const int t0 = k_lo / KT, nt = SETS ? walk.n : (k_hi > k_lo ? (k_hi + KT - 1) / KT - t0 : 0);
  auto tile_key = [&](int t) { return (SETS ? walk.at(t) : t0 + t) * KT; };

  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + kvh * p.k_sh;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + kvh * p.v_sh;
  const T* qrow = static_cast<const T*>(p.q) + b * p.q_sb + tok * p.q_sn + hq * p.q_sh;
  const T* dorow = static_cast<const T*>(p.dout) + b * p.do_sb + tok * p.do_sn + hq * p.do_sh;
  const T* orow = static_cast<const T*>(p.out) + b * p.o_sb + tok * p.o_sn + hq * p.o_sh;
  const int64_t stat = (static_cast<int64_t>(b) * p.h_q + hq) * p.n_q + tok;
  float lse = some ? p.lse[stat] : INFINITY;  // (no key: every weight 0)
  Frag qf[NC], dof[NC];
  float dsum = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = 16 * c + 8 * half;
    const bool in = some && e < p.d;
    qf[c] = in ? O::load(qrow + e) : O::zero();
    dof[c] = in ? O::load(dorow + e) : O::zero();
    const Frag of = in ? O::load(orow + e) : O::zero();
    dsum = O::dot(dof[c], of, dsum);
    if (p.out_low != nullptr) {
      const Frag lf = in ? O::load(static_cast<const T*>(p.out_low) + (orow - static_cast<const T*>(p.out)) + e) : O::zero();
      dsum = O::dot(dof[c], lf, dsum);
    }
  }
  dsum += other_half(dsum);
  if (real && half == 0 && kw == 0)
    p.stats[stat] = make_float4(lse, dsum, __int_as_float(lo), __int_as_float(hi));

  const int sc = tid % NCH, sr = tid / NCH;
  const bool chunk_ok = sc * E < p.d;
  const int64_t kst = p.k_sn * O::kEsize, vst = p.v_sn * O::kEsize;  // bytes of a row
  const uint32_t ks = static_cast<uint32_t>(kst), vs = static_cast<uint32_t>(vst);
  const uint32_t koff = chunk_ok ? sr * ks + sc * 16 : kNoChunk, voff = chunk_ok ? sr * vs + sc * 16 : kNoChunk;
  uint4 kreg[NP], vreg[NP];
  auto load_tile = [&](int t) {
    const int j0 = tile_key(t), left = n_keys - j0, db = p.d * O::kEsize;
    const auto kb = row_buffer(kbase + j0 * p.k_sn, left >= KT ? kAllBytes : static_cast<int>((left - 1) * kst) + db);
    const auto vb = row_buffer(vbase + j0 * p.v_sn, left >= KT ? kAllBytes : static_cast<int>((left - 1) * vst) + db);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      kreg[i] = row_load(kb, koff + i * RPP * ks);
      vreg[i] = row_load(vb, voff + i * RPP * vs);
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
  if (nt > 0) {
    load_tile(0);
    store_tile(0);
  }
  settle(qf);
  settle(dof);
  settle(lse);
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) load_tile(t + 1);
    const char* kt = lds + (t & 1) * 2 * TB + kw * 32 * NSUB * RB;
    const char* vt = kt + TB;
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const int k0 = tile_key(t) + (kw * NSUB + u) * 32;
      if ((k0 < hi_max && k0 + 32 > lo_min) || (SETS && k0 < a_max && k0 + 32 > a_min)) {
        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = O::mfma(O::template row_frag<RB>(kt, 32 * u, c, lane), qf[c], s);
          dp = O::mfma(O::template row_frag<RB>(vt, 32 * u, c, lane), dof[c], dp);
        }
        const int kl = k0 + 4 * half;
        const float dist = static_cast<float>(kl - pos), nlse = rule.b - lse;
        const bool whole = k0 >= lo_max && k0 + 32 <= hi_min;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 8 * (i >> 2) + (i & 3);
          float f;
          const float x = rule.z(p.rule, s[i], slope, dist + static_cast<float>(j), f);
          const float w = exp2_w(fmaf(x, rule.a, nlse)) * (dp[i] - dsum) * f;
          s[i] = w;
        }
        if (!whole) {
          const int a = in_branch(lo - kl), z = in_branch(hi - kl);
          if constexpr (SETS) {
            const int x = in_branch(sp.z - kl), y = in_branch(sp.w - kl);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int j = 8 * (i >> 2) + (i & 3);
              if (!((j >= a && j < z) || (j >= x && j < y))) s[i] = 0.0f;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int j = 8 * (i >> 2) + (i & 3);
              if (j < a || j >= z) s[i] = 0.0f;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const Frag df = O::pack(s, c);
#pragma unroll
          for (int i = 0; i < ND; ++i) acc[i] = O::mfma(O::template col_frag<RB>(kt, 32 * u + 16 * c, 32 * i, lane), df, acc[i]);
        }
      }
    }
    if (t + 1 < nt) store_tile((t + 1) & 1);
  }

  if constexpr (KW > 1) {  // the first of the waves that share rows adds up
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);
    if (kw > 0) {
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float4*>(sums + (wave * 32 + (lane & 31)) * PS + 32 * i + 8 * e + 4 * half) =
              make_float4(acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]);
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int y = 1; y < KW; ++y)
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 x = *reinterpret_cast<const float4*>(sums + ((wave + y) * 32 + (lane & 31)) * PS + 32 * i + 8 * e + 4 * half);
          acc[i][4 * e] += x.x;
          acc[i][4 * e + 1] += x.y;
          acc[i][4 * e + 2] += x.z;
          acc[i][4 * e + 3] += x.w;
        }
  }
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) worst = finite(acc[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, other_half(worst));
  const bool again = some && worst != 0.0f;
  T* dqrow = static_cast<T*>(p.dq) + ((static_cast<int64_t>(b) * p.n_q + tok) * p.h_q + hq) * p.d;
  if (real && !again) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dd = 32 * i + 8 * e + 4 * half;
        const float z = p.inv_scale * Rule<T, RULE>::kSlopeUnit;
        if (dd < p.d)
          O::store4(dqrow + dd, some ? acc[i][4 * e] * z : 0.0f, some ? acc[i][4 * e + 1] * z : 0.0f,
                    some ? acc[i][4 * e + 2] * z : 0.0f, some ? acc[i][4 * e + 3] * z : 0.0f);
      }
  }
  uint64_t todo = __ballot(again && half == 0);
  while (todo != 0) {
    const int src = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int a = lane_value(lo, src), z = lane_value(hi, src), ps = lane_value(pos, src);
    const float sl = lane_value(slope, src), ls = lane_value(lse, src), ds0 = lane_value(dsum, src);
    const T* qr = static_cast<const T*>(lane_ptr(qrow, src));
    const T* dr = static_cast<const T*>(lane_ptr(dorow, src));
    T* dst = const_cast<T*>(static_cast<const T*>(lane_ptr(dqrow, src)));
    float o[2] = {0.0f, 0.0f};
    auto add = [&](int from, int to) {
      for (int j0 = from; j0 < to; j0 += 64) {
        const int j = min(j0 + lane, to - 1);
        float f;
        const float x = score_x<T>(p.rule, row_dot(qr, kbase + j * p.k_sn, p.d), sl, static_cast<float>(j - ps), f);
        const float w = exp2_w(x - ls) * (row_dot(dr, vbase + j * p.v_sn, p.d) - ds0) * f;
        for (int t = 0; t < min(64, to - j0); ++t) {
          const float wt = lane_value(w, t);
          const T* kr = kbase + static_cast<int64_t>(j0 + t) * p.k_sn;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (lane + 64 * e < p.d) o[e] = fmaf(wt, ld(kr + lane + 64 * e), o[e]);
        }
      }
    };
    add(a, z);
    if constexpr (SETS) {  // (what the two share counts once)
      const int x = lane_value(sp.z, src), y = lane_value(sp.w, src);
      add(x, min(y, max(a, x)));
      add(max(x, z), y);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < p.d) O::store1(dst + lane + 64 * e, o[e] * p.inv_scale);
  }
}

// How dkv_kernel's waves are set: KG groups of 32 keys, RW waves that share a
// group's keys and take the rows in turn, row tiles of 32 NSUB rows a wave.
//
// bf16 at D = 128: dK and dV take 128 registers, so that K and V as operands (64
// more) would leave one wave on a SIMD, waiting for each of its loads; they lie in
// LDS instead (half as many LDS reads again), and the block has eight waves.
template <typename T, int D, int KG_, int RW_>
struct DkvShape {
  static constexpr int KG = KG_, RW = RW_, kWaves = KG * RW, kThr = 64 * kWaves;
  static constexpr bool kInLds = sizeof(T) == 2 && D == 128;
  static constexpr int NSUB = RW == 1 && sizeof(T) == 2 ? 2 : 1;
  static constexpr int QT = 32 * RW * NSUB, SG = QT / 32;
  static constexpr int RB = D * static_cast<int>(sizeof(T)), TB = QT * RB, KB = 32 * KG * RB, PS = D + 4;
  static constexpr size_t tiles = static_cast<size_t>(4) * TB, keys = kInLds ? static_cast<size_t>(2) * KB : 0;
  static constexpr size_t sums = static_cast<size_t>(RW - 1) * KG * 32 * PS * sizeof(float);
  static constexpr size_t lds = keys + tiles > sums ? keys + tiles : sums;
  // waves a SIMD must hold
  static constexpr int kPerSimd = sizeof(T) == 2 && (kWaves == 8 || lds <= 80 * 1024) ? 2 : 1;
};

template <typename T, int D, int RULE, int KG, int RW, int VIEW>
__global__ __launch_bounds__(64 * KG * RW, (DkvShape<T, D, KG, RW>::kPerSimd * 4) / (KG * RW) > 0
                                               ? (DkvShape<T, D, KG, RW>::kPerSimd * 4) / (KG * RW)
                                               : 1) void dkv_kernel(BwdParams p) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  using S = DkvShape<T, D, KG, RW>;
  constexpr bool SETS = VIEW == kTwo;
  constexpr int RB = S::RB, NCH = RB / 16, E = 16 / O::kEsize, QT = S::QT, NSUB = S::NSUB, SG = S::SG;
  constexpr int SW = sizeof(T) == 2 ? kWide : kNarrow;
  constexpr int NC = D / 16, ND = D / 32, TB = S::TB, NT = S::kThr, RPP = NT / NCH, NP = (QT + RPP - 1) / RPP;
  extern __shared__ __align__(16) char lds[];  // [K, V of the block's keys][2 buffers][Q, dO][TB]
  __shared__ __align__(16) float s_lse[2][QT], s_dsum[2][QT], s_slope[2][QT], s_pos[2][QT];
  __shared__ __align__(16) int s_lo[2][QT], s_hi[2][QT];
  __shared__ __align__(16) int s_x[2][SETS ? QT : 4], s_y[2][SETS ? QT : 4];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kg = wave / RW;
  int b, kvh, split, splits, tile, slot = 0;
  const bool planned = SETS && p.entries != nullptr;
  if (planned) {
    kvh = blockIdx.x % p.h_kv;
    const int4 entry = p.entries[blockIdx.x / p.h_kv];
    if (entry.x < 0) return;
    b = entry.x / p.key_tiles;
    tile = entry.x - b * p.key_tiles;
    split = entry.y;
    splits = entry.z;
    slot = entry.w;
  } else {
    const int nbh = p.batch * p.h_kv;
    const int bh = blockIdx.x % nbh;
    const int rest = blockIdx.x / nbh;
    splits = p.splits;
    split = rest % splits;
    tile = rest / splits;
    b = bh / p.h_kv;
    kvh = bh - b * p.h_kv;
  }
  const int n_keys = static_cast<int>(p.n), n_rows = static_cast<int>(p.n_q * p.g);
  const int kb0 = tile * 32 * KG;    // the block's keys
  const int kw0 = kb0 + kg * 32;     // the wave's
  const int key = kw0 + (lane & 31);
  const bool real = key < n_keys;
  const Rule<T, RULE> rule(p.rule);

  const T* krow = static_cast<const T*>(p.k) + b * p.k_sb + kvh * p.k_sh + static_cast<int64_t>(real ? key : 0) * p.k_sn;
  const T* vrow = static_cast<const T*>(p.v) + b * p.v_sb + kvh * p.v_sh + static_cast<int64_t>(real ? key : 0) * p.v_sn;
  char* keys = lds;
  char* bufs = lds + S::keys;
  Frag kf[S::kInLds ? 1 : NC], vf[S::kInLds ? 1 : NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = 16 * c + 8 * half;
    const bool in = real && e < p.d;
    if constexpr (S::kInLds) {
      if (rw == 0) {
        const int at = chunk_at<RB, SW>(kg * 32 + (lane & 31), 2 * c + half);
        *reinterpret_cast<uint4*>(keys + at) = in ? *reinterpret_cast<const uint4*>(krow + e) : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(keys + S::KB + at) = in ? *reinterpret_cast<const uint4*>(vrow + e) : make_uint4(0u, 0u, 0u, 0u);
      }
    } else {
      kf[c] = in ? O::load(krow + e) : O::zero();
      vf[c] = in ? O::load(vrow + e) : O::zero();
    }
  }

  // The row tiles that see some key of the block, in ascending order: lane x holds
  // the bounds of the x-th tile of 64.
  // (of parts, each takes every splits-th one: they are as long as each other
  // whatever the mask)
  const int t_end = (p.groups + SG - 1) / SG;
  const int4* bounds = p.bounds + static_cast<int64_t>(b) * p.groups * (SETS ? 2 : 1);
  int t_base = -64, t_seen = 0;
  uint64_t t_mask = 0;
  int4 bd[SG];
  int2 ba[SETS ? SG : 1];
  struct Pick {
    int tile;
    int lo_min[NSUB], hi_max[NSUB], lo_max[NSUB], hi_min[NSUB];  // of this wave's groups
    int a_min[NSUB], a_max[NSUB];
  };
  auto group_bounds = [&](int g) { return bounds[SETS ? 2 * g : g]; };
  auto seen_by = [&](const int4& x, int g) {  // whether the group's rows see some key of the block
    if (x.x < kb0 + 32 * KG && x.y > kb0) return true;
    if constexpr (SETS) {
      const int4 a = bounds[2 * g + 1];
      return a.x < kb0 + 32 * KG && a.y > kb0;
    }
    return false;
  };
  auto next_tile = [&](Pick& pk) {
    while (t_mask == 0) {
      t_base += 64;
      if (t_base >= t_end) {
        pk.tile = -1;
        return;
      }
      bool hit = false;
#pragma unroll
      for (int x = 0; x < SG; ++x) {
        const int g = (t_base + lane) * SG + x;
        const bool in = t_base + lane < t_end && g < p.groups;
        bd[x] = in ? group_bounds(g) : make_int4(0x7FFFFFFF, 0, 0, 0);
        hit |= bd[x].x < kb0 + 32 * KG && bd[x].y > kb0;
        if constexpr (SETS) {
          const int4 a = in ? bounds[2 * g + 1] : make_int4(0x7FFFFFFF, 0, 0, 0);
          ba[x] = make_int2(a.x, a.y);
          hit |= a.x < kb0 + 32 * KG && a.y > kb0;
        }
      }
      t_mask = __ballot(hit);
      if (splits > 1) {
        const int at = t_seen + __popcll(t_mask & ((uint64_t(1) << lane) - 1));
        t_seen += __popcll(t_mask);
        t_mask = __ballot(hit && static_cast<uint32_t>(at) % static_cast<uint32_t>(splits) == static_cast<uint32_t>(split));
      }
    }
    const int x = __builtin_ctzll(t_mask);
    t_mask &= t_mask - 1;
    pk.tile = t_base + x;
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      // (rw is the same for the whole wave)
      int4 mine = bd[u];
#pragma unroll
      for (int y = 1; y < RW; ++y)
        if (rw == y) mine = bd[y * NSUB + u];
      pk.lo_min[u] = lane_value(mine.x, x);
      pk.hi_max[u] = lane_value(mine.y, x);
      pk.lo_max[u] = lane_value(mine.z, x);
      pk.hi_min[u] = lane_value(mine.w, x);
      if constexpr (SETS) {
        int2 a = ba[u];
#pragma unroll
        for (int y = 1; y < RW; ++y)
          if (rw == y) a = ba[y * NSUB + u];
        pk.a_min[u] = lane_value(a.x, x);
        pk.a_max[u] = lane_value(a.y, x);
      }
    }
  };

  const int sc = tid % NCH, sr = tid / NCH;
  const bool chunk_ok = sc * E < p.d;
  // (the group's first head: 32-bit offsets step over a tile's tokens and the group's heads only)
  const T* qbase = static_cast<const T*>(p.q) + b * p.q_sb + kvh * p.g * p.q_sh;
  const T* dbase = static_cast<const T*>(p.dout) + b * p.do_sb + kvh * p.g * p.do_sh;
  const uint32_t qs = static_cast<uint32_t>(p.q_sn * O::kEsize), qh = static_cast<uint32_t>(p.q_sh * O::kEsize);
  const uint32_t ds = static_cast<uint32_t>(p.do_sn * O::kEsize), dh = static_cast<uint32_t>(p.do_sh * O::kEsize);
  uint4 qreg[NP], dreg[NP];
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  int2 st_set = make_int2(0, 0);
  float st_slope = 0.0f, st_pos = 0.0f;  // (positions count from the block's first key: past 2^24 a float holds no odd one)
  auto load_rows = [&](int t) {
    // offsets from the tile's first token
    const uint32_t tok0 = static_cast<uint32_t>(t * QT) / static_cast<uint32_t>(p.g);
    const auto qb = row_buffer(qbase + tok0 * p.q_sn, kAllBytes), db = row_buffer(dbase + tok0 * p.do_sn, kAllBytes);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t r = min(t * QT + min(sr + i * RPP, QT - 1), n_rows - 1);
      const uint32_t tok = r / static_cast<uint32_t>(p.g), h = r - tok * p.g;
      qreg[i] = row_load(qb, chunk_ok ? (tok - tok0) * qs + h * qh + sc * 16 : kNoChunk);
      dreg[i] = row_load(db, chunk_ok ? (tok - tok0) * ds + h * dh + sc * 16 : kNoChunk);
    }
    if (tid < QT) {
      const uint32_t r = min(t * QT + tid, n_rows - 1);
      const uint32_t tok = r / static_cast<uint32_t>(p.g), hq = kvh * p.g + r - tok * p.g;
      st = p.stats[(static_cast<int64_t>(b) * p.h_q + hq) * p.n_q + tok];
      if constexpr (SETS) {
        const int4 s = row_sets(p, b, tok);
        st_set = make_int2(s.z, s.w);
      }
      if constexpr (has_bias(RULE)) {
        st_slope = slope_of(p.rule, hq);
        st_pos = static_cast<float>(static_cast<int>(p.q_pos0 + tok) - kb0);
      }
    }
  };
  auto store_rows = [&](int t, int buf) {
    char* qt = bufs + buf * 2 * TB;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = sr + i * RPP;
      if (QT % RPP != 0 && row >= QT) break;
      const int at = chunk_at<RB, SW>(row, sc);
      *reinterpret_cast<uint4*>(qt + at) = qreg[i];
      *reinterpret_cast<uint4*>(qt + TB + at) = dreg[i];
    }
    if (tid < QT) {
      const bool in = t * QT + tid < n_rows;  // a row past the last one sees nothing
      s_lse[buf][tid] = in ? rule.b - st.x : -INFINITY;
      s_dsum[buf][tid] = st.y;
      s_lo[buf][tid] = in ? __float_as_int(st.z) : 0;
      s_hi[buf][tid] = in ? __float_as_int(st.w) : 0;
      if constexpr (SETS) {
        s_x[buf][tid] = in ? st_set.x : 0;
        s_y[buf][tid] = in ? st_set.y : 0;
      }
      if constexpr (has_bias(RULE)) {
        s_slope[buf][tid] = st_slope;
        s_pos[buf][tid] = st_pos;
      }
    }
  };

  f32x16 acck[ND], accv[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    acck[i] = f32x16{};
    accv[i] = f32x16{};
  }
  Pick cur, nx;
  next_tile(cur);
  if (cur.tile >= 0) {
    load_rows(cur.tile);
    store_rows(cur.tile, 0);
  }
  if constexpr (!S::kInLds) {
    settle(kf);
    settle(vf);
  }
  for (int t = 0; cur.tile >= 0; ++t) {
    __syncthreads();
    next_tile(nx);
    if (nx.tile >= 0) load_rows(nx.tile);
    const int buf = t & 1;
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      if ((cur.lo_min[u] >= kw0 + 32 || cur.hi_max[u] <= kw0) && (!SETS || cur.a_min[u] >= kw0 + 32 || cur.a_max[u] <= kw0)) continue;
      const int row0 = (rw * NSUB + u) * 32;
      const char* qt = bufs + buf * 2 * TB + row0 * RB;
      const char* dt = qt + TB;
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (S::kInLds) {
          const Frag kk = O::template row_frag<RB, SW>(keys, kg * 32, c, lane), vv = O::template row_frag<RB, SW>(keys + S::KB, kg * 32, c, lane);
          s = O::mfma(O::template row_frag<RB, SW>(qt, 0, c, lane), kk, s);
          dp = O::mfma(O::template row_frag<RB, SW>(dt, 0, c, lane), vv, dp);
        } else {
          s = O::mfma(O::template row_frag<RB, SW>(qt, 0, c, lane), kf[c], s);
          dp = O::mfma(O::template row_frag<RB, SW>(dt, 0, c, lane), vf[c], dp);
        }
      }
      const bool whole = cur.lo_max[u] <= kw0 && cur.hi_min[u] >= kw0 + 32 && cur.tile * QT + row0 + 32 <= n_rows;
      const float fkey = static_cast<float>(key - kb0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r0 = row0 + 8 * e + 4 * half;
        const float4 ls = *reinterpret_cast<const float4*>(&s_lse[buf][r0]);
        const float4 dd = *reinterpret_cast<const float4*>(&s_dsum[buf][r0]);
        float4 sl = make_float4(0.f, 0.f, 0.f, 0.f), ps = sl;
        if constexpr (has_bias(RULE)) {
          sl = *reinterpret_cast<const float4*>(&s_slope[buf][r0]);
          ps = *reinterpret_cast<const float4*>(&s_pos[buf][r0]);
        }
        const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dv[4] = {dd.x, dd.y, dd.z, dd.w};
        const float slv[4] = {sl.x, sl.y, sl.z, sl.w}, psv[4] = {ps.x, ps.y, ps.z, ps.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = 4 * e + x;
          float f;
          const float y = rule.z(p.rule, s[i], slv[x], fkey - psv[x], f);
          s[i] = exp2_w(fmaf(y, rule.a, lsv[x]));
          dp[i] = s[i] * (dp[i] - dv[x]) * f;
        }
        if (!whole) {
          const int my = in_branch(key);
          const int4 lo4 = *reinterpret_cast<const int4*>(&s_lo[buf][r0]);
          const int4 hi4 = *reinterpret_cast<const int4*>(&s_hi[buf][r0]);
          const int lov[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hiv[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
          int xv[4] = {0, 0, 0, 0}, yv[4] = {0, 0, 0, 0};
          if constexpr (SETS) {
            const int4 x4 = *reinterpret_cast<const int4*>(&s_x[buf][SETS ? r0 : 0]);
            const int4 y4 = *reinterpret_cast<const int4*>(&s_y[buf][SETS ? r0 : 0]);
            xv[0] = x4.x; xv[1] = x4.y; xv[2] = x4.z; xv[3] = x4.w;
            yv[0] = y4.x; yv[1] = y4.y; yv[2] = y4.z; yv[3] = y4.w;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const bool see = (my >= lov[x] && my < hiv[x]) || (SETS && my >= xv[x] && my < yv[x]);
            s[4 * e + x] = see ? s[4 * e + x] : 0.0f;
            dp[4 * e + x] = see ? dp[4 * e + x] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag pf = O::pack(s, c), df = O::pack(dp, c);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          accv[i] = O::mfma(O::template col_frag<RB, SW>(dt, 16 * c, 32 * i, lane), pf, accv[i]);
          acck[i] = O::mfma(O::template col_frag<RB, SW>(qt, 16 * c, 32 * i, lane), df, acck[i]);
        }
      }
    }
    if (nx.tile >= 0) store_rows(nx.tile, (t + 1) & 1);
    cur = nx;
  }

  if constexpr (RW > 1) {  // the first of the waves that share keys adds up, dK and then dV
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      f32x16(&acc)[ND] = which == 0 ? acck : accv;
      __syncthreads();
      if (rw > 0) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float4*>(sums + ((kg * (RW - 1) + rw - 1) * 32 + (lane & 31)) * S::PS + 32 * i + 8 * e + 4 * half) =
                make_float4(acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]);
      }
      __syncthreads();
      if (rw == 0) {
#pragma unroll
        for (int y = 0; y < RW - 1; ++y)
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 x = *reinterpret_cast<const float4*>(sums + ((kg * (RW - 1) + y) * 32 + (lane & 31)) * S::PS + 32 * i + 8 * e + 4 * half);
              acc[i][4 * e] += x.x;
              acc[i][4 * e + 1] += x.y;
              acc[i][4 * e + 2] += x.z;
              acc[i][4 * e + 3] += x.w;
            }
      }
    }
    if (rw > 0) return;
  }
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) worst = finite(acck[i][e]) && finite(accv[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, other_half(worst));
  const bool again = real && worst != 0.0f;
  const int64_t kid = (static_cast<int64_t>(b) * p.n + (real ? key : 0)) * p.h_kv + kvh;
  const int64_t kids = static_cast<int64_t>(p.batch) * p.n * p.h_kv;
  T* dkrow = static_cast<T*>(p.dk) + kid * p.d;
  T* dvrow = static_cast<T*>(p.dv) + kid * p.d;
  // where a key's parts go: by part and key, or (kTwo) by slot, head and key of the block
  auto part_at = [&](int64_t id, int key_) {
    if (planned) return ((static_cast<int64_t>(slot + split) * p.h_kv + kvh) * (32 * KG) + (key_ - kb0)) * D;
    return (split * kids + id) * D;
  };
  float* pk = splits > 1 ? p.part_k + part_at(kid, real ? key : kb0) : nullptr;
  float* pv = splits > 1 ? p.part_v + part_at(kid, real ? key : kb0) : nullptr;
  if (real && !again) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dd = 32 * i + 8 * e + 4 * half;
        if (dd >= p.d) continue;
        const float z = p.inv_scale * Rule<T, RULE>::kSlopeUnit;
        const float4 a = make_float4(acck[i][4 * e] * z, acck[i][4 * e + 1] * z, acck[i][4 * e + 2] * z, acck[i][4 * e + 3] * z);
        const float4 c = make_float4(accv[i][4 * e], accv[i][4 * e + 1], accv[i][4 * e + 2], accv[i][4 * e + 3]);
        if (splits > 1) {
          *reinterpret_cast<float4*>(pk + dd) = a;
          *reinterpret_cast<float4*>(pv + dd) = c;
        } else {
          O::store4(dkrow + dd, a.x, a.y, a.z, a.w);
          O::store4(dvrow + dd, c.x, c.y, c.z, c.w);
        }
      }
  }
  uint64_t todo = __ballot(again && half == 0);
  while (todo != 0) {  // this key's sums again, over the rows that see it
    const int src = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int kj = lane_value(key, src);
    const T* kr = static_cast<const T*>(lane_ptr(krow, src));
    const T* vr = static_cast<const T*>(lane_ptr(vrow, src));
    float ok[2] = {0.0f, 0.0f}, ov[2] = {0.0f, 0.0f};
    const T* qall = static_cast<const T*>(p.q) + b * p.q_sb;
    const T* dall = static_cast<const T*>(p.dout) + b * p.do_sb;
    int at = 0;  // tiles seen, as next_tile counts them
    for (int t = 0; t < t_end; ++t) {
      if (splits > 1) {
        bool hit = false;
        for (int x = t * SG; x < min((t + 1) * SG, p.groups); ++x) hit |= seen_by(group_bounds(x), x);
        if (!hit || at++ % splits != split) continue;
      }
      const int r_end = min(n_rows, (t + 1) * QT);
      for (int r0 = t * QT; r0 < r_end; r0 += 64) {
      const int r = r0 + lane;
      bool see = false;
      float w = 0.0f, ds = 0.0f;
      if (r < r_end) {
        const int tok = r / p.g, hq = kvh * p.g + r - tok * p.g;
        if constexpr (SETS) {
          const int4 sp = row_sets(p, b, tok);
          see = (kj >= sp.x && kj < sp.y) || (kj >= sp.z && kj < sp.w);
        } else {
          const int2 sp = row_span(p, b, tok);
          see = kj >= sp.x && kj < sp.y;
        }
        if (see) {
          const int64_t stat = (static_cast<int64_t>(b) * p.h_q + hq) * p.n_q + tok;
          const float sl = has_bias(RULE) ? slope_of(p.rule, hq) : 0.0f;
          float f;
          const float x = score_x<T>(p.rule, row_dot(qall + tok * p.q_sn + hq * p.q_sh, kr, p.d), sl,
                                           static_cast<float>(kj - (static_cast<int>(p.q_pos0) + tok)), f);
          const float4 rs = p.stats[stat];
          w = exp2_w(x - rs.x);
          ds = w * (row_dot(dall + tok * p.do_sn + hq * p.do_sh, vr, p.d) - rs.y) * f;
        }
      }
      uint64_t on = __ballot(see);
      while (on != 0) {
        const int x = __builtin_ctzll(on);
        on &= on - 1;
        const int rr = r0 + x, tok = rr / p.g, hq = kvh * p.g + rr - tok * p.g;
        const float wx = lane_value(w, x), dx = lane_value(ds, x);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (lane + 64 * e < p.d) {
            ov[e] = fmaf(wx, ld(dall + tok * p.do_sn + hq * p.do_sh + lane + 64 * e), ov[e]);
            ok[e] = fmaf(dx, ld(qall + tok * p.q_sn + hq * p.q_sh + lane + 64 * e), ok[e]);
          }
      }
      }
    }
    const int64_t id = (static_cast<int64_t>(b) * p.n + kj) * p.h_kv + kvh;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < p.d) {
        const int dd = lane + 64 * e;
        if (splits > 1) {
          p.part_k[part_at(id, kj) + dd] = ok[e] * p.inv_scale;
          p.part_v[part_at(id, kj) + dd] = ov[e];
        } else {
          O::store1(static_cast<T*>(p.dk) + id * p.d + dd, ok[e] * p.inv_scale);
          O::store1(static_cast<T*>(p.dv) + id * p.d + dd, ov[e]);
        }
      }
  }
}

// dk and dv from the parts, four features a thread, in part order.
template <typename T, int D>
__global__ __launch_bounds__(256) void dkv_join_kernel(BwdParams p) {
  const int per = p.d / 4;
  const int64_t kids = static_cast<int64_t>(p.batch) * p.n * p.h_kv;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= 2 * kids * per) return;
  const bool isv = t >= kids * per;
  const int64_t u = isv ? t - kids * per : t, kid = u / per;
  const int dd = static_cast<int>(u - kid * per) * 4;
  const float* part = isv ? p.part_v : p.part_k;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = 0; x < p.splits; ++x) {
    const float4 a = *reinterpret_cast<const float4*>(part + (x * kids + kid) * D + dd);
    s.x += a.x;
    s.y += a.y;
    s.z += a.z;
    s.w += a.w;
  }
  Op<T>::store4(static_cast<T*>(isv ? p.dv : p.dk) + kid * p.d + dd, s.x, s.y, s.z, s.w);
}

// kTwo: how many tiles of sg groups of rows see each block of keys.
[[maybe_unused]] __global__ __launch_bounds__(256) void plan_count_kernel(BwdParams p, int keys, int sg) {
  const int at = blockIdx.x, b = at / p.key_tiles, k0 = (at - b * p.key_tiles) * keys;
  const int tiles = (p.groups + sg - 1) / sg;
  const int4* bounds = p.bounds + static_cast<int64_t>(b) * p.groups * 2;
  __shared__ int s_sum[4];
  int n = 0;
  for (int t = threadIdx.x; t < tiles; t += 256) {
    bool hit = false;
    for (int g = t * sg; g < min((t + 1) * sg, p.groups); ++g) {
      const int4 x = bounds[2 * g], a = bounds[2 * g + 1];
      hit |= (x.x < k0 + keys && x.y > k0) || (a.x < k0 + keys && a.y > k0);
    }
    n += hit ? 1 : 0;
  }
  const int w = lane_value(wave_incl_scan(n), 63);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0)
    p.counts[at] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
}

// The blocks of dkv_kernel, by one block.  A slot is a block of keys, of one head, that runs at a
// time; share = what each of `slots` has to do on average.
//   h tiles > share   cut into parts of a tenth of the share (the more of them there are, the
//                     longer, up to a quarter: `extra` parts in all)
//   the others        whole, the longest first, so that the device's last blocks are short ones;
//                     where those of the last round would leave a good part of it idle they are cut
//                     until they fill it
// parts come after whole blocks (16001 rows that see 1000 keys back and 4 first ones, 16 / 4 heads,
// d = 128: dK and dV 640 us with parts first and as long as whole blocks, 525 so).
// At most key_blocks + most entries, most parts, 2 slots cut blocks.
constexpr int kPlan = 1024;  // (the rules are in ssa_cuts.h)
static_assert(kSorted == 2 * kPlan, "a thread ranks two blocks");
struct PlanSums {
  int64_t wave[kPlan / 64];
};
__device__ __forceinline__ int64_t plan_sum(int64_t x, PlanSums& s) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = x;
  __syncthreads();
  int64_t all = 0;
  for (int y = 0; y < kPlan / 64; ++y) all += s.wave[y];
  return all;
}
// Exclusive sums over the block's threads, and the whole block's.
__device__ __forceinline__ int plan_scan(int x, int (&s)[kPlan / 64], int& all) {
  const int incl = wave_incl_scan(x), wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s[wave] = incl;
  __syncthreads();
  int before = 0;
  all = 0;
  for (int y = 0; y < kPlan / 64; ++y) {
    if (y < wave) before += s[y];
    all += s[y];
  }
  return before + incl - x;
}

[[maybe_unused]] __global__ __launch_bounds__(kPlan) void plan_list_kernel(BwdParams p, int least, int slots, int most) {
  __shared__ PlanSums s_sums;
  __shared__ int s_scan[kPlan / 64];
  __shared__ __align__(16) int s_h[kSorted + 16];
  const int tid = threadIdx.x, N = p.key_blocks;
  const bool sorted = N <= kSorted;
  int64_t mine = 0;
  for (int x = tid; x < N; x += kPlan) {
    const int h = p.counts[x];
    mine += h;
    if (sorted) s_h[x] = h;
  }
  if (sorted && tid < 16) s_h[N + tid] = 0x7FFFFFFF;
  const int64_t total = plan_sum(mine, s_sums);
  const int64_t share = plan_share(total, slots, least);
  int64_t big = 0, n_big = 0;
  for (int x = tid; x < N; x += kPlan) {
    const int h = p.counts[x];
    if (h > share) {
      big += h;
      ++n_big;
    }
  }
  big = plan_sum(big << 24 | n_big, s_sums);  // (few are big: fewer than 2^24 of them, and tiles below 2^39)
  n_big = big & 0xFFFFFF;
  big >>= 24;
  const int P = plan_part(big, p.extra, least, share);
  // whole blocks of the last round
  const int n_one = N - static_cast<int>(n_big), left = plan_left(N, n_one, slots), n_whole = n_one - left;
  const bool cut_left = left > 0;
  int rank[kSorted / kPlan];
#pragma unroll
  for (int c = 0; c < kSorted / kPlan; ++c) {
    rank[c] = 0;
    const int x = c * kPlan + tid;
    if (!sorted || x >= N || s_h[x] > share) continue;
    const int h = s_h[x], top = static_cast<int>(share);
    int n = 0;
#pragma unroll 4
    for (int y = 0; y < N; y += 4) {  // (s_h is padded with blocks past any share)
      const int4 o = *reinterpret_cast<const int4*>(&s_h[y]);
      n += (o.x <= top && (o.x > h || (o.x == h && y < x))) + (o.y <= top && (o.y > h || (o.y == h && y + 1 < x))) +
           (o.z <= top && (o.z > h || (o.z == h && y + 2 < x))) + (o.w <= top && (o.w > h || (o.w == h && y + 3 < x)));
    }
    rank[c] = n;
  }
  int P2 = P;
  if (cut_left) {
    int64_t sum = 0;
#pragma unroll
    for (int c = 0; c < kSorted / kPlan; ++c) {
      const int x = c * kPlan + tid;
      if (x < N && s_h[x] <= share && rank[c] >= n_whole) sum += s_h[x];
    }
    sum = plan_sum(sum, s_sums);
    P2 = plan_left_part(sum, slots, least);
  }
  int at_part = 0, at_cut = 0, at_one = 0;
  for (int x0 = 0, c = 0; x0 < N; x0 += kPlan, ++c) {
    const int x = x0 + tid, h = x < N ? p.counts[x] : 0;
    const bool is_big = x < N && h > share;
    const int rk = sorted ? (c == 0 ? rank[0] : rank[1]) : 0;
    const bool is_left = cut_left && x < N && !is_big && rk >= n_whole;
    const int parts = is_big || is_left ? plan_parts(h, is_big ? P : P2) : 0;
    const int whole = x < N && !is_big && !is_left ? 1 : 0;
    int all_parts, all_cut, all_one;
    const int b_part = plan_scan(parts, s_scan, all_parts), b_cut = plan_scan(parts > 0 ? 1 : 0, s_scan, all_cut);
    const int b_one = plan_scan(whole, s_scan, all_one);
    if (whole) p.entries[sorted ? rk : at_one + b_one] = make_int4(x, 0, 1, 0);
    if (parts > 0) {
      const int from = at_part + b_part;
      // (a block in one part is whole: it needs no join)
      p.cut[1 + at_cut + b_cut] = make_int4(parts > 1 ? x : -1, parts, from, 0);
      for (int y = 0; y < parts; ++y) p.entries[n_whole + from + y] = make_int4(x, y, parts, from);
    }
    at_part += all_parts;
    at_cut += all_cut;
    at_one += all_one;
  }
  if (tid == 0) p.cut[0] = make_int4(at_cut, 0, 0, 0);
  for (int x = n_whole + at_part + tid; x < N + most; x += kPlan) p.entries[x] = make_int4(-1, 0, 0, 0);
}

// dk and dv of the cut blocks of keys, four features a thread, in part order, four parts' loads
// in flight.
template <typename T, int D>
__global__ __launch_bounds__(256) void dkv_two_join_kernel(BwdParams p, int keys) {
  const int per = p.d / 4, work = 2 * keys * per, pieces = (work + 255) / 256;
  const int items = p.cut[0].x * p.h_kv * pieces;
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int rest = it / pieces, x = (it - rest * pieces) * 256 + threadIdx.x;
    const int4 c = p.cut[1 + rest / p.h_kv];
    const int kvh = rest % p.h_kv;
    if (c.x < 0 || x >= work) continue;
    const int b = c.x / p.key_tiles, k0 = (c.x - b * p.key_tiles) * keys;
    const bool isv = x >= keys * per;
    const int u = isv ? x - keys * per : x, key = u / per, dd = (u - key * per) * 4;
    if (k0 + key >= p.n) continue;
    const int64_t step = static_cast<int64_t>(p.h_kv) * keys * D;
    const float* part = (isv ? p.part_v : p.part_k) + ((static_cast<int64_t>(c.z) * p.h_kv + kvh) * keys + key) * D + dd;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int y0 = 0; y0 < c.y; y0 += 4) {
      float4 a[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) a[y] = *reinterpret_cast<const float4*>(part + min(y0 + y, c.y - 1) * step);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (y0 + y >= c.y) continue;
        s.x += a[y].x;
        s.y += a[y].y;
        s.z += a[y].z;
        s.w += a[y].w;
      }
    }
    const int64_t id = (static_cast<int64_t>(b) * p.n + k0 + key) * p.h_kv + kvh;
    Op<T>::store4(static_cast<T*>(isv ? p.dv : p.dk) + id * p.d + dd, s.x, s.y, s.z, s.w);
  }
}

template <typename T, int D, int RULE, int KW, int VIEW>
int launch_dq(BwdParams& p, hipStream_t st) {
  const char* fn = "ssa_masked_attention_backward";
  const size_t bytes = dq_lds<T, D, KW>();
  if (int rc = reserve_lds(reinterpret_cast<const void*>(dq_kernel<T, D, RULE, KW, VIEW>), bytes + 1024, fn)) return rc;
  const int64_t blocks = ceil_div(p.n_q * p.g, kBlk / KW) * p.batch * p.h_kv;
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many rows", fn);
  dq_kernel<T, D, RULE, KW, VIEW><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), bytes, st>>>(p);
  return check_launch("ssa_masked_attention_backward dq");
}

template <typename T, int D, int RULE, int KG, int RW, int VIEW>
int launch_dkv(BwdParams& p, const TwoCut& cut, hipStream_t st) {
  const char* fn = "ssa_masked_attention_backward";
  using S = DkvShape<T, D, KG, RW>;
  if (int rc = reserve_lds(reinterpret_cast<const void*>(dkv_kernel<T, D, RULE, KG, RW, VIEW>), S::lds + (VIEW == kTwo ? 32 : 24) * S::QT * 2 + 1024, fn)) return rc;
  if (VIEW == kTwo && p.entries != nullptr) {
    // (parts of at least 128 rows, as of one interval)
    constexpr int least = S::QT < 128 ? 128 / S::QT : 1;
    const int64_t grid = static_cast<int64_t>(p.key_blocks + cut.most) * p.h_kv;
    if (grid > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many keys", fn);
    plan_count_kernel<<<dim3(static_cast<unsigned>(p.key_blocks)), dim3(256), 0, st>>>(p, 32 * KG, S::SG);
    plan_list_kernel<<<dim3(1), dim3(kPlan), 0, st>>>(p, least, cut.slots, cut.most);
    if (int rc = check_launch("ssa_masked_attention_backward plan")) return rc;
    dkv_kernel<T, D, RULE, KG, RW, VIEW><<<dim3(static_cast<unsigned>(grid)), dim3(S::kThr), S::lds, st>>>(p);
    if (int rc = check_launch("ssa_masked_attention_backward dkv")) return rc;
    dkv_two_join_kernel<T, D><<<dim3(1024), dim3(256), 0, st>>>(p, 32 * KG);
    return check_launch("ssa_masked_attention_backward join");
  }
  const int64_t nbh = static_cast<int64_t>(p.batch) * p.h_kv;
  const int64_t blocks = ceil_div(p.n, 32 * KG) * nbh * p.splits;
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many keys", fn);
  dkv_kernel<T, D, RULE, KG, RW, VIEW><<<dim3(static_cast<unsigned>(blocks)), dim3(S::kThr), S::lds, st>>>(p);
  if (int rc = check_launch("ssa_masked_attention_backward dkv")) return rc;
  if (p.splits > 1) {
    const int64_t work = 2 * nbh * p.n * (p.d / 4);
    dkv_join_kernel<T, D><<<dim3(static_cast<unsigned>(ceil_div(work, 256))), dim3(256), 0, st>>>(p);
    return check_launch("ssa_masked_attention_backward join");
  }
  return SSA_OK;
}

template <typename T, int D, int RULE, int VIEW>
int launch_bwd(BwdParams& p, const BwdCut& cut, const TwoCut& two, hipStream_t st) {
  int rc;
  if (most_kw<T, D>() >= 4 && cut.kw == 4)
    rc = launch_dq<T, D, RULE, most_kw<T, D>(), VIEW>(p, st);
  else
    rc = cut.kw >= 2 ? launch_dq<T, D, RULE, 2, VIEW>(p, st) : launch_dq<T, D, RULE, 1, VIEW>(p, st);
  if (rc) return rc;
  if constexpr (sizeof(T) == 2 && D == 128) {
    return cut.key_groups == 4 ? launch_dkv<T, D, RULE, 4, 2, VIEW>(p, two, st) : launch_dkv<T, D, RULE, 2, 2, VIEW>(p, two, st);
  } else {
    if constexpr (D == 64)
      if (cut.key_groups == 1) return launch_dkv<T, D, RULE, 1, 4, VIEW>(p, two, st);
    return cut.key_groups == 4 ? launch_dkv<T, D, RULE, 4, 1, VIEW>(p, two, st) : launch_dkv<T, D, RULE, 2, 2, VIEW>(p, two, st);
  }
}

template <typename T, int D, int VIEW>
int launch_rule(BwdParams& p, const BwdCut& cut, const TwoCut& two, hipStream_t st) {
  switch (rule_kind<T>(p.rule)) {
    case kPlain: return launch_bwd<T, D, kPlain, VIEW>(p, cut, two, st);
    case kCap: return launch_bwd<T, D, kCap, VIEW>(p, cut, two, st);
    case kBias: return launch_bwd<T, D, kBias, VIEW>(p, cut, two, st);
    case kFar:
      if constexpr (sizeof(T) == 2) return launch_bwd<T, D, kFar, VIEW>(p, cut, two, st);
  }
  return fail(SSA_ERR_UNSUPPORTED, "no kernel for this rule of scores");
}

}  // namespace
}  // namespace ssa
