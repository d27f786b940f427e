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
// Masked rows or keys that hold infinities or NaN: as in the forward, sums that
// end up other than finite are computed again pair by pair, visible pairs only.

#include <math.h>

#include "ssa_cuts.h"
#include "ssa_internal.h"
#include "ssa_tile.h"

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

// dkv_kernel's offsets of a tile's 128 packed rows, ceil(127 / g) tokens and g - 1 heads from
// the first one's, have to stay within its resource.
int check_group(const char* fn, const char* name, int dtype, int g, int d, int64_t sn, int64_t sh) {
  const int64_t e = dtype == SSA_DTYPE_F32 ? 4 : 2, room = kAllBytes / e - d - (126 + g) / g * sn;
  if (g > 1 && sh > room / (g - 1))
    return fail(SSA_ERR_UNSUPPORTED, "%s: the heads of a group of %s must lie within 2 GiB", fn, name);
  return SSA_OK;
}

// x (log2 units) and 1 - t^2 of a raw product, one pair at a time.
template <typename T>
__device__ __forceinline__ float score_x(const ScoreRule& r, float dot, float slope, float dist, float& factor) {
  if (sizeof(T) == 2 && r.cap == kSeries) return Rule<T, kFar>(r).z(r, dot, slope, dist, factor);
  return Rule<T, kBias>(r).z(r, dot, slope, dist, factor);
}

template <typename T>
__device__ __forceinline__ float row_dot(const T* a, const T* b, int d) {
  float s = 0.0f;
  for (int e = 0; e < d; e += 8) s = Op<T>::dot(Op<T>::load(a + e), Op<T>::load(b + e), s);
  return s;
}

__device__ __forceinline__ const void* lane_ptr(const void* x, int src) {
  const uint64_t u = reinterpret_cast<uint64_t>(x);
  return reinterpret_cast<const void*>(
      (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(u >> 32), src))) << 32) |
      static_cast<uint32_t>(lane_value(static_cast<int>(u & 0xFFFFFFFFu), src)));
}

// Waves of dq_kernel that may share rows: fp32 rows of 128 features fill the LDS with two.
template <typename T, int D>
constexpr int most_kw() {
  return sizeof(T) == 4 && D == 128 ? 2 : 4;
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

template <typename T, int D, int RULE, int KW>
__global__ __launch_bounds__(kThreads, (dq_lds<T, D, KW>() > 80 * 1024 || (sizeof(T) == 4 && D == 128) ? 1 : 2)) void dq_kernel(BwdParams p) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int RB = D * O::kEsize, NCH = RB / 16, E = 16 / O::kEsize;
  constexpr int KT = dq_keys<T, D, KW>();
  constexpr int NSUB = KT / (32 * KW), NC = D / 16, ND = D / 32, BR = kBlk / KW, PS = D + 4;
  constexpr int RPP = kThreads / NCH, NP = KT / RPP, TB = KT * RB;
  extern __shared__ __align__(16) char lds[];
  __shared__ int s_range[4][2];

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
  const int2 sp = real ? row_span(p, b, tok) : make_int2(0, 0);
  const int lo = sp.x, hi = sp.y;
  const bool some = real && hi > lo;
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const int lo_min = wave_min_i(some ? lo : 0x7FFFFFFF), hi_max = wave_max_i(some ? hi : 0);
  const int lo_max = wave_max_i(real ? lo : 0), hi_min = wave_min_i(real ? hi : 0x7FFFFFFF);
  if (lane == 0) {
    s_range[wave][0] = lo_min;
    s_range[wave][1] = hi_max;
    const int grp = tile * (BR / 32) + rw;
    if (kvh == 0 && kw == 0 && grp < p.groups) p.bounds[static_cast<int64_t>(b) * p.groups + grp] = make_int4(lo_min, hi_max, lo_max, hi_min);
  }
  __syncthreads();
  const int k_lo = __builtin_amdgcn_readfirstlane(min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0])));
  const int k_hi = __builtin_amdgcn_readfirstlane(max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1])));
  const int t0 = k_lo / KT, nt = k_hi > k_lo ? (k_hi + KT - 1) / KT - t0 : 0;

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
    const int j0 = (t0 + t) * KT, left = n_keys - j0, db = p.d * O::kEsize;
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
      const int k0 = (t0 + t) * KT + (kw * NSUB + u) * 32;
      if (k0 < hi_max && k0 + 32 > lo_min) {
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
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = 8 * (i >> 2) + (i & 3);
            if (j < a || j >= z) s[i] = 0.0f;
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
    for (int j0 = a; j0 < z; j0 += 64) {
      const int j = min(j0 + lane, z - 1);
      float f;
      const float x = score_x<T>(p.rule, row_dot(qr, kbase + j * p.k_sn, p.d), sl, static_cast<float>(j - ps), f);
      const float w = exp2_w(x - ls) * (row_dot(dr, vbase + j * p.v_sn, p.d) - ds0) * f;
      for (int t = 0; t < min(64, z - j0); ++t) {
        const float wt = lane_value(w, t);
        const T* kr = kbase + static_cast<int64_t>(j0 + t) * p.k_sn;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (lane + 64 * e < p.d) o[e] = fmaf(wt, ld(kr + lane + 64 * e), o[e]);
      }
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

template <typename T, int D, int RULE, int KG, int RW>
__global__ __launch_bounds__(64 * KG * RW, (DkvShape<T, D, KG, RW>::kPerSimd * 4) / (KG * RW) > 0
                                               ? (DkvShape<T, D, KG, RW>::kPerSimd * 4) / (KG * RW)
                                               : 1) void dkv_kernel(BwdParams p) {
  using O = Op<T>;
  using Frag = typename O::Frag;
  using S = DkvShape<T, D, KG, RW>;
  constexpr int RB = S::RB, NCH = RB / 16, E = 16 / O::kEsize, QT = S::QT, NSUB = S::NSUB, SG = S::SG;
  constexpr int SW = sizeof(T) == 2 ? kWide : kNarrow;
  constexpr int NC = D / 16, ND = D / 32, TB = S::TB, NT = S::kThr, RPP = NT / NCH, NP = (QT + RPP - 1) / RPP;
  extern __shared__ __align__(16) char lds[];  // [K, V of the block's keys][2 buffers][Q, dO][TB]
  __shared__ __align__(16) float s_lse[2][QT], s_dsum[2][QT], s_slope[2][QT], s_pos[2][QT];
  __shared__ __align__(16) int s_lo[2][QT], s_hi[2][QT];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave % RW, kg = wave / RW;
  const int nbh = p.batch * p.h_kv;
  const int bh = blockIdx.x % nbh;
  const int rest = blockIdx.x / nbh;
  const int split = rest % p.splits, tile = rest / p.splits;
  const int b = bh / p.h_kv, kvh = bh - b * p.h_kv;
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
  const int4* bounds = p.bounds + static_cast<int64_t>(b) * p.groups;
  int t_base = -64, t_seen = 0;
  uint64_t t_mask = 0;
  int4 bd[SG];
  struct Pick {
    int tile;
    int lo_min[NSUB], hi_max[NSUB], lo_max[NSUB], hi_min[NSUB];  // of this wave's groups
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
        bd[x] = t_base + lane < t_end && g < p.groups ? bounds[g] : make_int4(0x7FFFFFFF, 0, 0, 0);
        hit |= bd[x].x < kb0 + 32 * KG && bd[x].y > kb0;
      }
      t_mask = __ballot(hit);
      if (p.splits > 1) {
        const int at = t_seen + __popcll(t_mask & ((uint64_t(1) << lane) - 1));
        t_seen += __popcll(t_mask);
        t_mask = __ballot(hit && static_cast<uint32_t>(at) % static_cast<uint32_t>(p.splits) == static_cast<uint32_t>(split));
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
      if (cur.lo_min[u] >= kw0 + 32 || cur.hi_max[u] <= kw0) continue;
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
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const bool see = my >= lov[x] && my < hiv[x];
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
  float* pk = p.splits > 1 ? p.part_k + (split * kids + kid) * D : nullptr;
  float* pv = p.splits > 1 ? p.part_v + (split * kids + kid) * D : nullptr;
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
        if (p.splits > 1) {
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
      if (p.splits > 1) {
        bool hit = false;
        for (int x = t * SG; x < min((t + 1) * SG, p.groups); ++x) hit |= bounds[x].x < kb0 + 32 * KG && bounds[x].y > kb0;
        if (!hit || at++ % p.splits != split) continue;
      }
      const int r_end = min(n_rows, (t + 1) * QT);
      for (int r0 = t * QT; r0 < r_end; r0 += 64) {
      const int r = r0 + lane;
      bool see = false;
      float w = 0.0f, ds = 0.0f;
      if (r < r_end) {
        const int tok = r / p.g, hq = kvh * p.g + r - tok * p.g;
        const int2 sp = row_span(p, b, tok);
        see = kj >= sp.x && kj < sp.y;
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
        if (p.splits > 1) {
          p.part_k[(split * kids + id) * D + dd] = ok[e] * p.inv_scale;
          p.part_v[(split * kids + id) * D + dd] = ov[e];
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

template <typename T, int D, int RULE, int KW>
int launch_dq(BwdParams& p, hipStream_t st) {
  const char* fn = "ssa_masked_attention_backward";
  const size_t bytes = dq_lds<T, D, KW>();
  if (int rc = reserve_lds(reinterpret_cast<const void*>(dq_kernel<T, D, RULE, KW>), bytes + 1024, fn)) return rc;
  const int64_t blocks = ceil_div(p.n_q * p.g, kBlk / KW) * p.batch * p.h_kv;
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many rows", fn);
  dq_kernel<T, D, RULE, KW><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), bytes, st>>>(p);
  return check_launch("ssa_masked_attention_backward dq");
}

template <typename T, int D, int RULE, int KG, int RW>
int launch_dkv(BwdParams& p, hipStream_t st) {
  const char* fn = "ssa_masked_attention_backward";
  using S = DkvShape<T, D, KG, RW>;
  if (int rc = reserve_lds(reinterpret_cast<const void*>(dkv_kernel<T, D, RULE, KG, RW>), S::lds + 24 * S::QT * 2 + 1024, fn)) return rc;
  const int64_t nbh = static_cast<int64_t>(p.batch) * p.h_kv;
  const int64_t blocks = ceil_div(p.n, 32 * KG) * nbh * p.splits;
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many keys", fn);
  dkv_kernel<T, D, RULE, KG, RW><<<dim3(static_cast<unsigned>(blocks)), dim3(S::kThr), S::lds, st>>>(p);
  if (int rc = check_launch("ssa_masked_attention_backward dkv")) return rc;
  if (p.splits > 1) {
    const int64_t work = 2 * nbh * p.n * (p.d / 4);
    dkv_join_kernel<T, D><<<dim3(static_cast<unsigned>(ceil_div(work, 256))), dim3(256), 0, st>>>(p);
    return check_launch("ssa_masked_attention_backward join");
  }
  return SSA_OK;
}

template <typename T, int D, int RULE>
int launch_bwd(BwdParams& p, const BwdCut& cut, hipStream_t st) {
  int rc;
  if (most_kw<T, D>() >= 4 && cut.kw == 4)
    rc = launch_dq<T, D, RULE, most_kw<T, D>()>(p, st);
  else
    rc = cut.kw >= 2 ? launch_dq<T, D, RULE, 2>(p, st) : launch_dq<T, D, RULE, 1>(p, st);
  if (rc) return rc;
  if constexpr (sizeof(T) == 2 && D == 128) {
    return cut.key_groups == 4 ? launch_dkv<T, D, RULE, 4, 2>(p, st) : launch_dkv<T, D, RULE, 2, 2>(p, st);
  } else {
    if constexpr (D == 64)
      if (cut.key_groups == 1) return launch_dkv<T, D, RULE, 1, 4>(p, st);
    return cut.key_groups == 4 ? launch_dkv<T, D, RULE, 4, 1>(p, st) : launch_dkv<T, D, RULE, 2, 2>(p, st);
  }
}

template <typename T, int D>
int launch_rule(BwdParams& p, const BwdCut& cut, hipStream_t st) {
  switch (rule_kind<T>(p.rule)) {
    case kPlain: return launch_bwd<T, D, kPlain>(p, cut, st);
    case kCap: return launch_bwd<T, D, kCap>(p, cut, st);
    case kBias: return launch_bwd<T, D, kBias>(p, cut, st);
    case kFar:
      if constexpr (sizeof(T) == 2) return launch_bwd<T, D, kFar>(p, cut, st);
  }
  return fail(SSA_ERR_UNSUPPORTED, "no kernel for this rule of scores");
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

extern "C" int ssa_masked_attention_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q, int64_t q_pos0, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
    int64_t v_sn, int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes, const void* out,
    const void* out_low, int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "ssa_masked_attention_backward";
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
  const BwdCut l = bwd_cut(dtype, batch, n, n_q, h_q, h_kv, d);
  if (workspace == nullptr || workspace_bytes < l.bytes)
    return fail(SSA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", fn, l.bytes,
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
  if (l.splits > 1) {
    p.part_k = reinterpret_cast<float*>(ws + l.part);
    p.part_v = p.part_k + static_cast<int64_t>(l.splits) * batch * n * h_kv * (d <= 64 ? 64 : 128);
  }
  hipStream_t st = as_stream(stream);
  if (dtype == SSA_DTYPE_F32) return d <= 64 ? launch_rule<float, 64>(p, l, st) : launch_rule<float, 128>(p, l, st);
  return d <= 64 ? launch_rule<uint16_t, 64>(p, l, st) : launch_rule<uint16_t, 128>(p, l, st);
}
