// The kernels of a paged step (ssa_paged.hip says what they do): appending, few rows, the
// joins, and how a call's cut and score rule choose among them.
#pragma once

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

// One row of new keys or values as 8-bit codes with a scale, by 16 lanes of eight features each.
// scale = max |x| / 127 (int8) or / 448 (e4m3), rounded to fp32; a code is the nearest to x / scale.
// The quotient is rounded to odd before it is rounded to the code, so that no second rounding
// moves one that lies next to a border: fp32's nearest is off the exact quotient by less than half
// a step, x - y scale is exact in one fma, and of the two floats around an inexact quotient the
// odd one rounds to fewer bits as the quotient does.  Rows below 2^-100 are zeros (the remainder
// would leave fp32); a row that holds an infinity or NaN has the scale NaN.
__device__ __forceinline__ float odd_quotient(float x, float scale) {
  const float y = x / scale, r = fmaf(-y, scale, x);
  uint32_t u = __float_as_uint(y);
  if (r != 0.0f && (u & 1u) == 0) u += (r < 0.0f) == (x < 0.0f) ? 1 : -1;
  return __uint_as_float(u);
}

template <typename T>
__device__ __forceinline__ void append_row(const DenseParams& p, int64_t t) {
  const int64_t total = p.n_q * p.h_kv;
  const int c = static_cast<int>(t & 15);
  const int64_t at = t >> 4;
  // (the 16 lanes of a row stay together: their reductions want all of them)
  const bool isv = at >= total;
  const int64_t row = isv ? at - total : at;
  bool on = at < 2 * total;
  const int tok = on ? static_cast<int>(row / p.h_kv) : 0, h = on ? static_cast<int>(row - static_cast<int64_t>(tok) * p.h_kv) : 0;
  const int b = on ? sequence_of(p, tok) : -1;
  on = on && b >= 0 && b < p.batch;
  Seq s{0, 0, 0};
  if (on) s = paged_seq(p, b);
  on = on && tok >= s.first && tok < s.first + s.m;
  const int j = s.len - s.m + tok - s.first;
  int pg = 0;
  if (on) {
    pg = p.table[b * p.table_stride + (j >> p.page_log2)];
    if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.num_pages)) {
      if (p.error_flag != nullptr) atomicOr(p.error_flag, 1);
      on = false;
    }
  }
  const bool mine = on && c * 8 < p.d;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (mine) {
    const T* src = static_cast<const T*>(isv ? p.v_new : p.k_new) + tok * (isv ? p.vn_st : p.kn_st) +
                   h * (isv ? p.vn_sh : p.kn_sh) + c * 8;
    if constexpr (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(src);
      const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(v[e] << 16);
        x[2 * e + 1] = __uint_as_float(v[e] & 0xFFFF0000u);
      }
    } else {
      const float4 w = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
      x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
      x[4] = y.x; x[5] = y.y; x[6] = y.z; x[7] = y.w;
    }
  }
  float most = 0.0f;
  int odd = 0;  // an element that is not finite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    most = fmaxf(most, fabsf(x[e]));
    odd |= finite(x[e]) ? 0 : 1;
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor(most, o, 64));
    odd |= __shfl_xor(odd, o, 64);
  }
  if (!on) return;
  float scale = odd != 0 ? __uint_as_float(0x7FC00000u) : (most < 7.888609052210118e-31f ? 0.0f : most / (p.e4m3 ? 448.0f : 127.0f));
  const int64_t r = j & ((1 << p.page_log2) - 1);
  if (mine) {
    uint32_t w[2] = {0u, 0u};
    if (scale > 0.0f) {  // (not NaN)
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = odd_quotient(x[e], scale);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (p.e4m3) {
          int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
          v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], v, true);
          w[i] = static_cast<uint32_t>(v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = max(-127, min(127, static_cast<int>(rintf(y[4 * i + e]))));
            w[i] |= (static_cast<uint32_t>(v) & 0xFFu) << (8 * e);
          }
        }
      }
    }
    uint8_t* dst = static_cast<uint8_t*>(const_cast<void*>(isv ? p.v : p.k)) + pg * (isv ? p.v_sb : p.k_sb) +
                   r * (isv ? p.v_sn : p.k_sn) + h * (isv ? p.v_sh : p.k_sh) + c * 8;
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
  if (c == 0) {
    float* dst = const_cast<float*>(isv ? p.v_scale : p.k_scale) + pg * (isv ? p.vs_sb : p.ks_sb) +
                 r * (isv ? p.vs_sn : p.ks_sn) + h * (isv ? p.vs_sh : p.ks_sh);
    *dst = scale;
  }
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

// kTwo: the 32-key tiles that a sequence's new tokens see.
__device__ __forceinline__ Tiles seq_tiles(const DenseParams& p, const Seq& s) {
  return seen_tiles(s.len - s.m, s.len, p.window, p.sinks, 32);
}

template <typename T, int D, int RULE, int VIEW = kOne, typename S = T>
__device__ __forceinline__ void few_rows(const DenseParams& p, const int block, char* lds) {
  constexpr bool SETS = VIEW == kTwo, HELD = !std::is_same_v<S, T>;
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int RB = D * O::kEsize, NCH = RB / 16, E = 16 / O::kEsize;
  constexpr int NC = D / 16, ND = D / 32, TB = 32 * RB;
  constexpr int RPW = 64 / NCH, NP = 32 / RPW;  // rows a wave's load instruction covers; loads of a tile
  constexpr int PS = D + 4;                     // floats of a row of partial sums
  // lds: [4 waves][K, V][TB], then [4][32][PS] sums
  __shared__ float s_m[4][kFew], s_l[4][kFew];
  __shared__ int s_bad[4][kFew];
  __shared__ uint64_t s_kin[SETS ? kDrafts : 1];
  __shared__ int s_depth[SETS ? kDrafts : 1];
  __shared__ __align__(16) float s_scale[HELD ? 4 : 1][HELD ? 2 : 1][HELD ? 32 : 1];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = block % p.h_kv;
  const int rest = block / p.h_kv;
  const int split = rest % p.splits, b = rest / p.splits;
  const Seq sq = paged_seq(p, b);
  const int R = sq.m * p.g;
  if (R == 0 || R > p.few_rows) return;
  const int cached = sq.len - sq.m;
  // the part's keys, and of kTwo its tiles t_begin .. t_end of those that the rows see
  int k_begin = 0, k_end = sq.len, t_begin = 0, t_end = 0, part_x[2] = {0, 0}, part_y[2] = {0, 0};
  Tiles walk{0, 0, 0, 0};
  int first_a = 0, from = 0;  // keys below the one and from the other on are seen by some row
  if constexpr (SETS) {
    walk = seq_tiles(p, sq);
    const int per = static_cast<int>(p.split_len / 32);
    t_begin = static_cast<int>(min(static_cast<int64_t>(split) * per, static_cast<int64_t>(walk.n)));
    t_end = min(t_begin + per, walk.n);
    if (t_begin >= t_end) return;  // (a part past the sequence's tiles, which the join does not read)
    part_x[0] = (walk.x0 + min(t_begin, walk.n1)) * 32;
    part_y[0] = (walk.x0 + min(t_end, walk.n1)) * 32;
    part_x[1] = (walk.y0 + max(t_begin - walk.n1, 0)) * 32;
    part_y[1] = (walk.y0 + max(t_end - walk.n1, 0)) * 32;
    if (p.window > 0) {
      first_a = min(p.sinks, max(sq.len - p.window, 0));
      from = max(cached + 1 - p.window, 0);
    }
  } else {
    k_begin = static_cast<int>(min(split * p.split_len, static_cast<int64_t>(sq.len)));
    k_end = static_cast<int>(min((split + 1) * p.split_len, static_cast<int64_t>(sq.len)));
    if (k_begin >= k_end) return;  // (a part past the sequence, which the join does not read)
  }
  const KeyRows<T, true, S> rows = key_rows<T, true, S>(p, b, kvh, sq.first, cached);

  const int rr = lane & 31;
  const bool real = rr < R;
  const int tok = real ? rr / p.g : 0;
  const int hq = kvh * p.g + (real ? rr - tok * p.g : 0);
  int pos = cached + tok;
  Sees see{0, 0, 0, 0, cached, 0};
  const bool tree = SETS && p.parents != nullptr;
  if constexpr (SETS) {
    uint64_t kin = 0;
    if (tree) {
      int depth;
      const uint64_t all = draft_kin(p, sq.first, sq.m, cached, depth);
      if (lane < kDrafts) {  // (each wave the same)
        s_kin[lane] = all;
        s_depth[lane] = depth;
      }
      wave_lds_sync();
      kin = s_kin[tok];
      pos = cached + s_depth[tok];
    }
    see = paged_sees(p, pos, cached, kin);
  }
  // the keys that every row sees
  const int lo_max = SETS && p.window > 0 ? max(sq.len - p.window, 0) : 0, hi_min = tree ? cached : cached + 1;
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
  // HELD: a load covers eight rows of one page, eight lanes a row (16 codes each, or 8 of 64 features)
  constexpr int CB = D / 8, NW = CB / 4;  // bytes and words of a lane's chunk
  uint4 kreg[HELD ? 4 : NP], vreg[HELD ? 4 : NP];
  const int my_row = lane >> 3, my_at = (lane & 7) * CB;
  const uint32_t ks8 = static_cast<uint32_t>(rows.k_sn), vs8 = static_cast<uint32_t>(rows.v_sn);
  // kTwo: a key of the sequence that stands for key j where j is looked up, one that some row sees
  // (or a new one, whose page the table has too)
  auto seen_key = [&](int j) { return min(j >= first_a ? max(j, from) : j, k_end - 1); };
  int outside = 0;  // whether a page of a tile was outside the pool
  float scale_reg = 1.0f;  // HELD: of K's key lane, from lane 32 on of V's key lane - 32
  auto pages_at = [&](int k0) {
    if constexpr (SETS) return k0 >= 0 ? rows.entry_of(seen_key(k0 + rr)) : 0;
    return k0 < k_end ? rows.entry_of(min(k0 + rr, k_end - 1)) : 0;
  };
  auto load_tile = [&](int k0, int entry) {
    const int pg = rows.noted(entry, outside);
    if constexpr (HELD) {
      const int j = seen_key(k0 + rr);
      scale_reg = rows.is_new(j) ? 1.0f : rows.scale_of(half != 0, pg, j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t page = lane_value(pg, 8 * i), r0 = (k0 + 8 * i) & rows.page_mask;
        const auto kb = row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes);
        const auto vb = row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes);
        const uint32_t ko = my_row * ks8 + my_at, vo = my_row * vs8 + my_at;
        if constexpr (CB == 16) {
          if (p.d & 8) {  // (rows of 8 bytes more than 16s: a chunk's second half may lie past the row)
            const bool a = my_at < p.d, b = my_at + 8 < p.d;
            const uint4 k0_ = Codes<uint16_t>::load(kb, a ? ko : kNoChunk), k1_ = Codes<uint16_t>::load(kb, b ? ko + 8 : kNoChunk);
            const uint4 v0_ = Codes<uint16_t>::load(vb, a ? vo : kNoChunk), v1_ = Codes<uint16_t>::load(vb, b ? vo + 8 : kNoChunk);
            kreg[i] = make_uint4(k0_.x, k0_.y, k1_.x, k1_.y);
            vreg[i] = make_uint4(v0_.x, v0_.y, v1_.x, v1_.y);
          } else {
            kreg[i] = row_load(kb, my_at < p.d ? ko : kNoChunk);
            vreg[i] = row_load(vb, my_at < p.d ? vo : kNoChunk);
          }
        } else {
          kreg[i] = Codes<uint16_t>::load(kb, my_at < p.d ? ko : kNoChunk);
          vreg[i] = Codes<uint16_t>::load(vb, my_at < p.d ? vo : kNoChunk);
        }
      }
      return;
    }
    if constexpr (!HELD)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = sr + i * RPW;
      const T *kr, *vr;
      rows.in_page(__shfl(pg, r, 64), SETS ? seen_key(k0 + r) : min(k0 + r, k_end - 1), kr, vr);
      kreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(kr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
      vreg[i] = chunk_ok ? *reinterpret_cast<const uint4*>(vr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
    }
  };

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{};
  float mref = -INFINITY, lsum = 0.0f;

  // kOne: x is the tile's first key; kTwo: its number, of which a wave takes every fourth
  constexpr int STEP = SETS ? 4 : 128;
  const int x_end = SETS ? t_end : k_end;
  auto key_at = [&](int x) { return SETS ? (x < x_end ? walk.at(x) * 32 : -1) : x; };
  int x = SETS ? t_begin + wave : k_begin + 32 * wave;
  int pg = pages_at(key_at(x));
  if (x < x_end) load_tile(key_at(x), pg);
  pg = pages_at(key_at(x + STEP));
  settle(qf);
  for (; x < x_end; x += STEP) {
    const int k0 = key_at(x);
    if constexpr (!HELD) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int at = chunk_at<RB>(sr + i * RPW, sc);
        *reinterpret_cast<uint4*>(kt + at) = kreg[i];
        *reinterpret_cast<uint4*>(vt + at) = vreg[i];
      }
    } else {
      if (k0 + 32 > min(rows.new_from, k_end)) {  // (rows without a key may hold a code for NaN, which a weight of 0 does not silence)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + 8 * i + my_row >= min(rows.new_from, k_end)) vreg[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      auto put = [&](auto kind) {
        constexpr bool E4M3 = decltype(kind)::value;
        constexpr int W = sizeof(T) == 2 ? 2 : 1;  // words of codes that make 16 bytes of T
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t kw[4] = {kreg[i].x, kreg[i].y, kreg[i].z, kreg[i].w}, vw[4] = {vreg[i].x, vreg[i].y, vreg[i].z, vreg[i].w};
#pragma unroll
          for (int c = 0; c < NW / W; ++c) {
            const int at = chunk_at<RB>(8 * i + my_row, (lane & 7) * (NW / W) + c);
            *reinterpret_cast<uint4*>(kt + at) = Codes<T>::template widen<E4M3>(kw[W * c], kw[(W * c + 1) & 3]);
            *reinterpret_cast<uint4*>(vt + at) = Codes<T>::template widen<E4M3>(vw[W * c], vw[(W * c + 1) & 3]);
          }
        }
      };
      if (rows.e4m3)
        put(std::true_type());
      else
        put(std::false_type());
      s_scale[wave][half][rr] = scale_reg;
      if (k0 + 32 > rows.new_from) {  // the call's own rows, as they are given
        wave_lds_sync();  // (over what other lanes have put there)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int r = sr + i * RPW, j = seen_key(k0 + r);
          if (!rows.is_new(j)) continue;
          const T *kr, *vr;
          rows.new_rows(j, kr, vr);
          const int at = chunk_at<RB>(r, sc);
          *reinterpret_cast<uint4*>(kt + at) = chunk_ok ? *reinterpret_cast<const uint4*>(kr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(vt + at) = chunk_ok ? *reinterpret_cast<const uint4*>(vr + sc * E) : make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
    wave_lds_sync();
    if (x + STEP < x_end) load_tile(key_at(x + STEP), pg);
    pg = pages_at(key_at(x + 2 * STEP));
    f32x16 s = f32x16{};
#pragma unroll
    for (int c = 0; c < NC; ++c) s = O::mfma(O::template row_frag<RB>(kt, 0, c, lane), qf[c], s);
    const int kl = k0 + 4 * half;
    const float dist = static_cast<float>(kl - pos);
    float top = Rule<T, RULE>::kHidden;
    if constexpr (!SETS) {
      const int z = min(pos + 1, k_end) - kl;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 8 * (i >> 2) + (i & 3);
        s[i] = rule.z(p.rule, s[i], slope, dist + static_cast<float>(j));
        if (j >= z) s[i] = Rule<T, RULE>::kHidden;
        top = rule.better(top, s[i]);
      }
    } else {
      if constexpr (HELD)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 f = *reinterpret_cast<const float4*>(&s_scale[wave][0][8 * e + 4 * half]);
          s[4 * e] *= f.x;
          s[4 * e + 1] *= f.y;
          s[4 * e + 2] *= f.z;
          s[4 * e + 3] *= f.w;
        }
      if (has_bias(RULE) && tree && k0 + 32 > cached) {  // (drafts lie at cached + depth)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = kl + 8 * (i >> 2) + (i & 3), n = j - cached;
          const int at = n < 0 ? j : cached + s_depth[min(n, kDrafts - 1)];
          s[i] = rule.z(p.rule, s[i], slope, static_cast<float>(at - pos));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = rule.z(p.rule, s[i], slope, dist + static_cast<float>(8 * (i >> 2) + (i & 3)));
      }
      if (k0 < lo_max || k0 + 32 > hi_min) {
        const int a = in_branch(see.lo - kl), z = in_branch(see.hi - kl), y = in_branch(see.a_hi - kl);
        const uint32_t kin = kin_word(see.kin, k0 - cached) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 8 * (i >> 2) + (i & 3);
          if (!((j >= a && j < z) || j < y || (kin >> j & 1u) != 0)) s[i] = Rule<T, RULE>::kHidden;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = rule.better(top, s[i]);
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
    if constexpr (HELD)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 f = *reinterpret_cast<const float4*>(&s_scale[wave][HELD ? 1 : 0][8 * e + 4 * half]);
        s[4 * e] *= f.x;
        s[4 * e + 1] *= f.y;
        s[4 * e + 2] *= f.z;
        s[4 * e + 3] *= f.w;
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Frag pf = O::pack(s, c);
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[i] = O::mfma(O::template col_frag<RB>(vt, 16 * c, 32 * i, lane), pf, acc[i]);
    }
    wave_lds_sync();
  }
  rows.report(outside);

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
  // whether the part holds a key that token t sees
  auto sees_of = [&](int t) { return paged_sees(p, cached + (tree ? s_depth[SETS ? t : 0] : t), cached, tree ? s_kin[SETS ? t : 0] : 0); };
  auto here_of = [&](int t) {
    if constexpr (!SETS) return k_begin < min(k_end, cached + t + 1);
    const Sees w = sees_of(t);
    return w.any(part_x[0], part_y[0]) || w.any(part_x[1], part_y[1]);
  };
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
        p.part_ml[pr * 2] = here_of(t) && m == -INFINITY ? -3.0e38f : m;
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
    const int t = r / p.g, h = kvh * p.g + r - t * p.g, ps = cached + (tree ? s_depth[SETS ? t : 0] : t);
    const float sl = has_bias(RULE) ? slope_of(p.rule, h) : 0.0f;
    float o[4], m, l;
    const T* qr = static_cast<const T*>(p.q) + (sq.first + t) * p.q_sn + h * p.q_sh;
    if constexpr (SETS) {
      m = -INFINITY;
      l = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = 0.0f;
#pragma unroll
      for (int y = 0; y < 2; ++y)
        exact_keys<T, S, true>(rows, p.rule, sees_of(t), qr, p.d, part_x[y], min(part_y[y], sq.len), sl, ps, tree ? s_depth : nullptr,
                               o, m, l);
    } else {
      exact_row<T, true>(rows, p.rule, qr, p.d, k_begin, min(k_end, ps + 1), sl, ps, o, m, l);
    }
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
      p.part_ml[pr * 2] = here_of(t) && m == -INFINITY ? -3.0e38f : m;
      p.part_ml[pr * 2 + 1] = l;
    }
  }
}

// few_rows for at most 16 rows of one or two new tokens over pages of 8 bits, bf16 queries.  Widening the codes, 1.5
// instructions a code, is most of the work beside memory's, so that the rest is kept small and
// more waves share a SIMD (two of few_rows do, whose tiles of bf16 fill the LDS): the LDS
// holds codes, widened as they are read, and 16x16x32 products, whose 16 columns spend half the
// softmax that 32 do.  A product's contraction takes the features in the order in which 16 bytes a
// lane bring them, and Q is loaded in that order too; V is transposed by its reads
// (ds_read_b64_tr_b8).  The call's own rows,
// which have no codes yet, are added one by one at the end, by one wave of the last part, wherever
// they lie.
// 64 sequences of 8191 cached tokens, 32 / 8 heads, int8: 233 to 240 us, 4.8 to 4.6 TB/s of codes and scales;
// ragged ones end at unlike times.  ssa_cuts.h's codes_call has both kernels' times.
constexpr int kCols = 16;
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 16 codes (8 of rows of at most 64) at a lane's and the wave's offset.
template <int D>
__device__ __forceinline__ uint4 load_codes(__amdgpu_buffer_rsrc_t rows, uint32_t lane_at, int at) {
  if constexpr (D == 128) {
    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rows, static_cast<int>(lane_at), at, 0);
    return make_uint4(x.x, x.y, x.z, x.w);
  } else {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rows, static_cast<int>(lane_at), at, 0);
    return make_uint4(x.x, x.y, 0u, 0u);
  }
}

template <int D, int RULE>
__device__ __forceinline__ void few_codes(const DenseParams& p, const int block, char* lds) {
  using T = uint16_t;
  using S = uint8_t;
  using O = Op<T>;
  using Frag = typename O::Frag;
  constexpr int NS = D / 32, NH = D / 64, NF = D / 16;  // products of a score, a lane's loads of a row, tiles of features
  constexpr int CB = 32 * D, PS = D + 4;
  // lds: [4 waves][K, V][codes], then [4][16][PS] sums
  __shared__ float s_m[4][kCols], s_l[4][kCols];
  __shared__ int s_bad[4][kCols];
  __shared__ uint64_t s_kin[kDrafts];
  __shared__ int s_depth[kDrafts];
  __shared__ __align__(16) float s_scale[4][2][32];

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = block % p.h_kv, rest = block / p.h_kv;
  const int split = rest % p.splits, b = rest / p.splits;
  const Seq sq = paged_seq(p, b);
  const int R = sq.m * p.g;
  if (R == 0 || R > kCols) return;
  const int cached = sq.len - sq.m;
  const Tiles walk = seq_tiles(p, sq);
  const int per = static_cast<int>(p.split_len / 32);
  const int t_begin = static_cast<int>(min(static_cast<int64_t>(split) * per, static_cast<int64_t>(walk.n)));
  const int t_end = min(t_begin + per, walk.n);
  if (t_begin >= t_end) return;  // (a part past the sequence's tiles, which the join does not read)
  const int part_x[2] = {(walk.x0 + min(t_begin, walk.n1)) * 32, (walk.y0 + max(t_begin - walk.n1, 0)) * 32};
  const int part_y[2] = {(walk.x0 + min(t_end, walk.n1)) * 32, (walk.y0 + max(t_end - walk.n1, 0)) * 32};
  const int first_a = p.window > 0 ? min(p.sinks, max(sq.len - p.window, 0)) : 0;
  const int from = p.window > 0 ? max(cached + 1 - p.window, 0) : 0;
  const KeyRows<T, true, S> rows = key_rows<T, true, S>(p, b, kvh, sq.first, cached);

  const bool real = n < R;
  const int tok = real ? n / p.g : 0;
  const int hq = kvh * p.g + (real ? n - tok * p.g : 0);
  const bool tree = p.parents != nullptr;
  int pos = cached + tok;
  uint64_t kin = 0;
  if (tree) {
    int depth;
    const uint64_t all = draft_kin(p, sq.first, sq.m, cached, depth);
    if (lane < kDrafts) {  // (each wave the same)
      s_kin[lane] = all;
      s_depth[lane] = depth;
    }
    wave_lds_sync();
    kin = s_kin[tok];
    pos = cached + s_depth[tok];
  }
  const Sees see = paged_sees(p, pos, cached, kin);
  const int lo_max = p.window > 0 ? max(sq.len - p.window, 0) : 0, hi_min = min(rows.new_from, tree ? cached : cached + 1);
  const Rule<T, RULE> rule(p.rule);
  const float slope = has_bias(RULE) && real ? slope_of(p.rule, hq) : 0.0f;
  const T* qrow = static_cast<const T*>(p.q) + (sq.first + tok) * p.q_sn + hq * p.q_sh;
  auto feature = [&](int s) { return 64 * (s >> 1) + 16 * quad + 8 * (s & 1); };  // of product s, this lane's first
  Frag qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = real && feature(s) < p.d ? O::load(qrow + feature(s)) : O::zero();

  char* kt = lds + wave * 2 * CB;
  char* vt = kt + CB;
  // (the banks of a tile's rows: 16-byte chunk c of row r lies at chunk c ^ f(r))
  auto chunk = [&](int r, int c) { return r * D + ((c ^ (D == 128 ? r & 7 : (r >> 2) & 3)) << 4); };
  auto seen_key = [&](int j) { return min(j >= first_a ? max(j, from) : j, sq.len - 1); };
  // tiles of new keys alone are left out: they have no codes
  auto key_at = [&](int x) { return x < t_end ? walk.at(x) * 32 : 0x7FFFFFFF; };
  const int codes_end = min(rows.new_from, sq.len);
  const int my_row = lane >> 3, my_at = (lane & 7) * (D / 8), key32 = lane & 31;
  const uint32_t ko = my_at < p.d ? my_row * static_cast<uint32_t>(rows.k_sn) + my_at : kNoChunk;
  const uint32_t vo = my_at < p.d ? my_row * static_cast<uint32_t>(rows.v_sn) + my_at : kNoChunk;
  uint4 kreg[4], vreg[4];
  float scale_reg = 1.0f;  // of K's key lane, from lane 32 on of V's key lane - 32
  auto find = [&](int k0) { return k0 < codes_end ? rows.entry_of(seen_key(k0 + key32)) : 0; };
  auto load = [&](int k0, int entry) {
    const int pg = rows.checked(entry);
    const int j = seen_key(k0 + key32);
    scale_reg = j < codes_end ? rows.scale_of(lane >= 32, pg, j) : 1.0f;
    auto fetch = [&](int i, __amdgpu_buffer_rsrc_t kb, __amdgpu_buffer_rsrc_t vb, int ks, int vs) {
      kreg[i] = load_codes<D>(kb, ko, ks);
      vreg[i] = load_codes<D>(vb, vo, vs);
    };
    if (rows.page_mask >= 31) {  // (one page holds the tile)
      const int64_t page = lane_value(pg, 0), r0 = k0 & rows.page_mask;
      const auto kb = row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes);
      const auto vb = row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) fetch(i, kb, vb, 8 * i * static_cast<int>(rows.k_sn), 8 * i * static_cast<int>(rows.v_sn));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t page = lane_value(pg, 8 * i), r0 = (k0 + 8 * i) & rows.page_mask;
        fetch(i, row_buffer(rows.k + page * rows.k_sb + r0 * rows.k_sn, kAllBytes),
              row_buffer(rows.v + page * rows.v_sb + r0 * rows.v_sn, kAllBytes), 0, 0);
      }
    }
  };
  auto put = [&](char* tile, const uint4 (&reg)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      char* at = tile + chunk(8 * i + my_row, my_at >> 4) + (my_at & 15);
      if constexpr (D == 128)
        *reinterpret_cast<uint4*>(at) = reg[i];
      else
        *reinterpret_cast<uint2*>(at) = make_uint2(reg[i].x, reg[i].y);
    }
  };

  const int vr = 16 * (n >> 3) + 4 * quad + ((n >> 1) & 3);
  const int k_base = chunk(n, quad), v_base = chunk(vr, 0) + 8 * (n & 1);

  f32x4 acc[NF];
#pragma unroll
  for (int i = 0; i < NF; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float mref = -INFINITY, lsum = 0.0f;
  auto rescale = [&](float top) {  // moves the reference to at least top
    const float mn = fmaxf(mref, top);
    const float alpha = mref == mn ? 1.0f : exp2_w(mref - mn);
    mref = mn;
    lsum *= alpha;
#pragma unroll
    for (int i = 0; i < NF; ++i) acc[i] *= alpha;
  };

  int x = t_begin + wave;
  int entry = find(key_at(x));
  if (key_at(x) < codes_end) load(key_at(x), entry);
  entry = find(key_at(x + 4));
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    settle(qf[s].v.x);
    settle(qf[s].v.y);
    settle(qf[s].v.z);
    settle(qf[s].v.w);
  }
  auto walk_tiles = [&](auto kind) {
    constexpr bool E4M3 = decltype(kind)::value;
    for (; key_at(x) < codes_end; x += 4) {
      const int k0 = key_at(x);
      // (addresses that differ by an exclusive or are formed anew: kept, they take twelve registers)
      const int k_at = in_branch(k_base), v_at = in_branch(v_base);
      if (k0 + 32 > codes_end) {  // (rows without a key may hold a code for NaN, which a weight of 0 does not silence)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + 8 * i + my_row >= codes_end) vreg[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      put(kt, kreg);
      put(vt, vreg);
      s_scale[wave][lane >> 5][key32] = scale_reg;
      wave_lds_sync();
      if (key_at(x + 4) < codes_end) load(key_at(x + 4), entry);
      entry = find(key_at(x + 8));
      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const uint4 k = *reinterpret_cast<const uint4*>(kt + (k_at ^ (h << 6)) + 16 * D * u);
          const uint4 a = Codes<T>::template widen<E4M3>(k.x, k.y), c = Codes<T>::template widen<E4M3>(k.z, k.w);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, qf[2 * h].v), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c), __builtin_bit_cast(bf16x8, qf[2 * h + 1].v), s[u], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);  // (widened any earlier, the codes take the registers of a wave)
        }
      }
      const int kl = k0 + 4 * quad;  // key of register 0
      float top = Rule<T, RULE>::kHidden;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 f = *reinterpret_cast<const float4*>(&s_scale[wave][0][16 * u + 4 * quad]);
        const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = rule.z(p.rule, s[u][r] * fs[r], slope, static_cast<float>(kl + 16 * u + r - pos));
      }
      if (k0 < lo_max || k0 + 32 > hi_min) {  // (new keys come later)
        const int a = in_branch(see.lo - kl), z = in_branch(min(see.hi, rows.new_from) - kl), y = in_branch(min(see.a_hi, rows.new_from) - kl);
        const uint32_t kin = rows.new_from < sq.len ? 0u : kin_word(see.kin, k0 - cached) >> (4 * quad);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * u + r;
            if (!((j >= a && j < z) || j < y || (kin >> j & 1u) != 0)) s[u][r] = Rule<T, RULE>::kHidden;
          }
        if (has_bias(RULE) && tree && rows.new_from >= sq.len && k0 + 32 > cached) {  // (drafts that the pages hold lie at cached + depth)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = kl + 16 * u + r - cached;
              if (j >= 0 && j < kDrafts && (kin >> (16 * u + r) & 1u) != 0)
                s[u][r] += slope * (fabsf(static_cast<float>(cached + j - pos)) - fabsf(static_cast<float>(cached + s_depth[j] - pos)));
            }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = rule.better(top, s[u][r]);
      top = rule.better(top, __shfl_xor(top, 16, 64));
      top = fmaf(rule.better(top, __shfl_xor(top, 32, 64)), rule.a, rule.b);
      if (__ballot(top > mref + 8.0f) != 0) rescale(top);
      const float nref = rule.b - (mref == -INFINITY ? 0.0f : mref);
      uint32_t pk[4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 f = *reinterpret_cast<const float4*>(&s_scale[wave][1][16 * u + 4 * quad]);
        const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = exp2_w(fmaf(s[u][r], rule.a, nref));
          lsum += s[u][r];
          s[u][r] *= fs[r];
        }
        pk[2 * u] = O::pack2(s[u][0], s[u][1]);
        pk[2 * u + 1] = O::pack2(s[u][2], s[u][3]);
      }
      const uint4 pf = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      // lane i of a quad's 16 reads 8 bytes of the quad's keys 4 quad + {0..3, 16..19}, the (i / 2)-th,
      // and gets feature i of all eight
      typedef int v2i __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) v2i* lds_v2i;
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const v2i c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(vt + (v_at ^ (i << 4))));
        const uint4 a = Codes<T>::template widen<E4M3>(static_cast<uint32_t>(c.x), static_cast<uint32_t>(c.y));
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, pf), acc[i], 0, 0, 0);
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
      }
      wave_lds_sync();
    }
  };
  if (rows.e4m3)
    walk_tiles(std::true_type());
  else
    walk_tiles(std::false_type());

  // the call's own rows, as they are given
  if (t_end == walk.n && rows.new_from < sq.len && wave == 3) {
    for (int i = 0; i < sq.m; ++i) {
      const int j = cached + i;
      const T *kr, *vr;
      rows.new_rows(j, kr, vr);
      float dot = 0.0f;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (feature(s) < p.d) dot = O::dot(qf[s], O::load(kr + feature(s)), dot);
      dot += __shfl_xor(dot, 16, 64);
      dot += __shfl_xor(dot, 32, 64);
      const bool on = real && see.key(j);
      const int at = tree ? cached + s_depth[i] : j;
      const float sc = fmaf(rule.z(p.rule, dot, slope, static_cast<float>(at - pos)), rule.a, rule.b);
      if (on) rescale(sc);
      const float w = on ? exp2_w(sc - (mref == -INFINITY ? 0.0f : mref)) : 0.0f;
      lsum += quad == 0 ? w : 0.0f;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int c = 16 * f + 4 * quad;
        if (c >= p.d || !on) continue;
        const uint2 v = *reinterpret_cast<const uint2*>(vr + c);
        acc[f][0] = fmaf(w, __uint_as_float(v.x << 16), acc[f][0]);
        acc[f][1] = fmaf(w, __uint_as_float(v.x & 0xFFFF0000u), acc[f][1]);
        acc[f][2] = fmaf(w, __uint_as_float(v.y << 16), acc[f][2]);
        acc[f][3] = fmaf(w, __uint_as_float(v.y & 0xFFFF0000u), acc[f][3]);
      }
    }
  }

  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  float worst = finite(lsum) ? 0.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) worst = finite(acc[i][e]) ? worst : 1.0f;
  worst = fmaxf(worst, __shfl_xor(worst, 16, 64));
  worst = fmaxf(worst, __shfl_xor(worst, 32, 64));
  if (quad == 0) {
    s_m[wave][n] = mref;
    s_l[wave][n] = lsum;
    s_bad[wave][n] = worst != 0.0f;
  }
  __syncthreads();  // every wave is past its tiles: their LDS holds the sums now
  float* sums = reinterpret_cast<float*>(lds);
  if (real) {
#pragma unroll
    for (int i = 0; i < NF; ++i)
      *reinterpret_cast<float4*>(sums + (wave * kCols + n) * PS + 16 * i + 4 * quad) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  }
  __syncthreads();
  const int64_t part_row = (static_cast<int64_t>(b) * p.h_kv + kvh) * kFew;
  const int quads = p.d / 4;
  auto sees_of = [&](int t) { return paged_sees(p, cached + (tree ? s_depth[t] : t), cached, tree ? s_kin[t] : 0); };
  // whether the part holds a key that token t sees: of its tiles those with codes, of the last part
  // the call's own rows too
  const int own = t_end == walk.n && codes_end < sq.len ? sq.len : 0;
  auto here_of = [&](int t) {
    const Sees w = sees_of(t);
    return w.any(part_x[0], min(part_y[0], codes_end)) || w.any(part_x[1], min(part_y[1], codes_end)) || w.any(codes_end, own);
  };
  for (int e = tid; e < R * quads; e += kThreads) {
    const int r = e / quads, dd = (e - r * quads) * 4;
    if (s_bad[0][r] | s_bad[1][r] | s_bad[2][r] | s_bad[3][r]) continue;
    const float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float ref = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float a = exp2_w(s_m[y][r] - ref);
      const float4 w = *reinterpret_cast<const float4*>(sums + (y * kCols + r) * PS + dd);
      l = fmaf(a, s_l[y][r], l);
      o.x = fmaf(a, w.x, o.x);
      o.y = fmaf(a, w.y, o.y);
      o.z = fmaf(a, w.z, o.z);
      o.w = fmaf(a, w.w, o.w);
    }
    const int t = r / p.g, h = kvh * p.g + r - t * p.g;
    if (p.splits > 1) {
      const int64_t pr = split * p.part_rows + part_row + r;
      *reinterpret_cast<float4*>(p.part_o + pr * D + dd) = o;
      if (dd == 0) {
        // (a part whose visible keys all scored -inf says so by a finite m)
        p.part_ml[pr * 2] = here_of(t) && m == -INFINITY ? -3.0e38f : m;
        p.part_ml[pr * 2 + 1] = l;
      }
    } else {
      const float inv = 1.0f / l;
      O::store4(static_cast<T*>(p.out) + (sq.first + t) * p.o_sn + h * p.o_sh + dd, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
  }
  for (int r = wave; r < R; r += 4) {  // rows to compute again, key by key
    if (!(s_bad[0][r] | s_bad[1][r] | s_bad[2][r] | s_bad[3][r])) continue;
    const int t = r / p.g, h = kvh * p.g + r - t * p.g, ps = cached + (tree ? s_depth[t] : t);
    const float sl = has_bias(RULE) ? slope_of(p.rule, h) : 0.0f;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    const T* qr = static_cast<const T*>(p.q) + (sq.first + t) * p.q_sn + h * p.q_sh;
#pragma unroll
    for (int y = 0; y < 3; ++y)
      exact_keys<T, S, true>(rows, p.rule, sees_of(t), qr, p.d, y < 2 ? part_x[y & 1] : codes_end,
                             y < 2 ? min(part_y[y & 1], codes_end) : own, sl, ps, tree ? s_depth : nullptr, o, m, l);
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
      p.part_ml[pr * 2] = here_of(t) && m == -INFINITY ? -3.0e38f : m;
      p.part_ml[pr * 2 + 1] = l;
    }
  }
}

// Everything of a call in one launch: blocks of many rows (the longest) first, then
// few rows, then the blocks that append.  KW 0: no sequence has many rows (KW -1: none more than
// 16 of them, over pages of 8 bits); its call may
// have no second launch, so that the blocks of no rows stand here (beside dense_rows they
// cost 2048 rows behind 30720 cached 12%: 1215 to 1350 us).
template <typename T, int D, int KW>
constexpr int paged_per_cu() {
  if constexpr (KW > 0) return rows_per_cu<T, D, KW>();
  if constexpr (KW < 0) return 3;
  return sizeof(T) == 2 || D == 64 ? 2 : 1;
}

template <typename T, int D, int RULE, int KW, bool FRESH, int VIEW, typename S>
__global__ __launch_bounds__(kThreads, (paged_per_cu<T, D, KW>())) void paged_kernel(DenseParams rows, DenseParams few, int row_blocks,
                                                                                     int few_blocks, int copy_blocks) {
  extern __shared__ __align__(16) char lds[];
  const int w = blockIdx.x;
  if (w < row_blocks) {
    if constexpr (KW > 0) dense_rows<T, D, true, RULE, KW, FRESH, VIEW, S>(rows, w, lds);
  } else if (w < row_blocks + few_blocks) {
    if constexpr (KW < 0)
      few_codes<D, RULE>(few, w - row_blocks, lds);
    else
      few_rows<T, D, RULE, VIEW, S>(few, w - row_blocks, lds);
  } else if (KW > 0 || w < row_blocks + few_blocks + copy_blocks) {
    const int64_t t = static_cast<int64_t>(w - row_blocks - few_blocks) * kAppend + threadIdx.x;
    for (int i = 0; i < kAppend; i += kThreads) {
      if constexpr (std::is_same_v<S, T>)
        append_chunk<T>(few, t + i);
      else
        append_row<T>(few, t + i);
    }
  } else {
    if constexpr (KW <= 0) no_rows<T>(few, w - row_blocks - few_blocks - copy_blocks);
  }
}

// The parts of few-row sequences: `per` waves a row (1, 4 or 16 of the block's 16),
// each with every per-th part, eight parts' loads in flight; their sums meet in LDS.
constexpr int kJoinWaves = 16, kAtOnce = 8;

template <typename T, int D, int VIEW>
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
  const int64_t keys = VIEW == kTwo ? 32 * static_cast<int64_t>(seq_tiles(p, sq).n) : sq.len;
  const int parts = on ? static_cast<int>(min(static_cast<int64_t>(p.splits), ceil_div(keys, p.split_len))) : 0;
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
template <typename T, int D, int VIEW>
__global__ __launch_bounds__(kJoinWaves * 64) void paged_join_kernel(DenseParams rows, DenseParams few, int few_blocks,
                                                                          int join_blocks, int most_rows, int per) {
  if (static_cast<int>(blockIdx.x) < few_blocks)
    few_join<T, D, VIEW>(few, blockIdx.x, most_rows, per);
  else if (static_cast<int>(blockIdx.x) >= join_blocks)
    no_rows<T>(few, blockIdx.x - join_blocks);
  else
    dense_join<T, D>(rows, static_cast<int64_t>(blockIdx.x - few_blocks) * kJoinWaves + (threadIdx.x >> 6));
}

template <typename T, int D, int RULE, int KW, bool FRESH, int VIEW, typename S>
int launch_paged(DenseParams& p, const PagedPlan& l, bool zero_rows, char* ws, hipStream_t st) {
  const char* fn = "ssa_paged_step";
  constexpr bool HELD = !std::is_same_v<S, T>;
  const auto kernel = paged_kernel<T, D, RULE, KW, FRESH, VIEW, S>;
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
  if constexpr (KW < 0) bytes = static_cast<size_t>(4) * kCols * (D + 4) * sizeof(float);  // (more than V's codes take)
  if (int rc = reserve_lds(reinterpret_cast<const void*>(kernel), bytes + (VIEW == kTwo ? 8192 : 4096), fn)) return rc;
  const int64_t rblocks = static_cast<int64_t>(l.row_tiles) * p.h_kv * r.splits;
  const int64_t fblocks = static_cast<int64_t>(p.batch) * p.h_kv * f.splits;
  // pieces that a thread appends: 16 bytes, or an eighth of a wave's quarter of a row's codes
  const int64_t chunks = p.k_new == nullptr ? 0 : 2 * p.n_q * p.h_kv * (HELD ? 16 : p.d / (16 / static_cast<int>(sizeof(T))));
  const int most = static_cast<int>(p.max_new * p.g < kFew ? p.max_new * p.g : kFew);
  const int per = f.splits <= 8 ? 1 : (f.splits <= 32 ? 4 : 16);  // waves a row: one round of loads, or 16 waves
  const int64_t few_join_blocks = f.splits > 1 ? ceil_div(static_cast<int64_t>(p.batch) * p.h_kv * most, kJoinWaves / per) : 0;
  const int64_t join_blocks = few_join_blocks + (l.row_tiles > 0 && r.splits > 1 ? ceil_div(r.part_rows, kJoinWaves) : 0);
  const bool zero_here = zero_rows && KW <= 0 && join_blocks == 0;
  const int64_t second = join_blocks + (zero_rows && !zero_here ? ceil_div(p.n_q, kJoinWaves * 64) : 0);
  if (second > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many sequences", fn);
  const int64_t cblocks = ceil_div(chunks, kAppend);
  const int64_t blocks = rblocks + fblocks + cblocks + (zero_here ? ceil_div(p.n_q, kThreads) : 0);
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), bytes, st>>>(
      r, f, static_cast<int>(rblocks), static_cast<int>(fblocks), static_cast<int>(cblocks));
  if (int rc = check_launch("ssa_paged_step")) return rc;
  if (second > 0) {
    paged_join_kernel<T, D, VIEW><<<dim3(static_cast<unsigned>(second)), dim3(kJoinWaves * 64), 0, st>>>(
        r, f, static_cast<int>(few_join_blocks), static_cast<int>(join_blocks), most, per);
    return check_launch("ssa_paged_step join");
  }
  return SSA_OK;
}

// The kernel for a call's cut and score rule.
template <typename T, int D, int RULE, int VIEW, typename S>
int launch_kw(DenseParams& p, const PagedPlan& l, bool zero, char* ws, hipStream_t st) {
  if constexpr (!std::is_same_v<S, T> && sizeof(T) == 2)
    if (codes_call(SSA_DTYPE_BF16, SSA_DTYPE_I8, p.max_new, p.g, p.d)) return launch_paged<T, D, RULE, -1, false, VIEW, S>(p, l, zero, ws, st);
  if (l.row_tiles == 0) return launch_paged<T, D, RULE, 0, false, VIEW, S>(p, l, zero, ws, st);
  // Where a good part of the keys are the call's own rows, their tiles are read as
  // contiguous ones (four prompts of 1000 tokens, 32 / 8 heads: 117 to 81 us); the
  // branch costs the pages' tiles 16% (2048 tokens behind 30720: 1220 to 1410).  Pages of
  // 8 bits hold nothing of the call's own rows yet: their tiles always have a way of their own.
  constexpr bool HELD = !std::is_same_v<S, T>;
  const bool fresh = HELD || (p.k_new != nullptr && 3 * p.max_new >= p.max_len);
  auto go = [&](auto kw) {
    constexpr int KW = decltype(kw)::value;
    if constexpr (!HELD)
      if (!fresh) return launch_paged<T, D, RULE, KW, false, VIEW, S>(p, l, zero, ws, st);
    return launch_paged<T, D, RULE, KW, true, VIEW, S>(p, l, zero, ws, st);
  };
  if constexpr (most_kw<T, D>() >= 4)
    if (l.row_kw == 4) return go(std::integral_constant<int, 4>());
  if (l.row_kw == 2) return go(std::integral_constant<int, 2>());
  return go(std::integral_constant<int, 1>());
}

template <typename T, int D, int VIEW, typename S = T>
int launch_rule(DenseParams& p, const PagedPlan& l, bool zero, char* ws, hipStream_t st) {
  switch (rule_kind<T>(p.rule)) {
    case kPlain: return launch_kw<T, D, kPlain, VIEW, S>(p, l, zero, ws, st);
    case kCap: return launch_kw<T, D, kCap, VIEW, S>(p, l, zero, ws, st);
    case kBias: return launch_kw<T, D, kBias, VIEW, S>(p, l, zero, ws, st);
    case kFar:
      if constexpr (sizeof(T) == 2) return launch_kw<T, D, kFar, VIEW, S>(p, l, zero, ws, st);
  }
  return fail(SSA_ERR_UNSUPPORTED, "no kernel for this rule of scores");
}

}  // namespace
}  // namespace ssa
