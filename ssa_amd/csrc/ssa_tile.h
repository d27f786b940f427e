// Matrix-core tiles of the dense attention kernels (ssa_masked.hip,
// ssa_masked_bwd.hip, ssa_paged.hip): operand fragments, the LDS tile layout and
// the score rule they share.
//
// One layout serves every product.  A wave works on 32 "columns" (query rows,
// or keys in the dK/dV kernel) of a 32x32 MFMA: lane l holds column l % 32, and
// accumulator register r holds row 8 (r / 4) + 4 (l / 32) + r % 4.  A product's
// contraction may visit its index in any order as long as both operands use the
// same one, so the registers of a score tile are the next product's B operand as
// they stand: registers 8c .. 8c + 7 are the 16 rows
//   16 c + 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11}
// and only the A operand (read from LDS, by columns) follows that order.  No
// score moves between lanes.
//
// LDS tiles are [rows][D] with 16-byte chunks swizzled: chunk c of row r lies at
// chunk c ^ f(r).  The LDS serves 16 lanes of a 16-byte read and 32 of an 8-byte one
// at a time, from 64 banks.  Free of conflicts (kWide) is
//   f = 4 (r % 4) + (r / 4) % 4          rows of 256 bytes and more
//   f = 4 ((r / 2) % 2) + (r / 4) % 4    rows of 128 bytes, two to the banks' span
// for row fragments (one chunk of 16 rows) and column fragments (four chunks of four
// rows, ds_read_b64_tr_b16) alike.  kNarrow, f = 2 (r % 4) + (r / 4) % 2, reads both in
// twice the cycles but moves only three bits, so that one address serves more chunks
// by its offset.  The dK/dV kernel of bf16, whose LDS is the busiest, gains from the
// wide one (backward over 8192 x 8192, 32 heads, d 128: 4020 to 3780 us; d 64: alike);
// with it the forward spills at d 128 (1125 to 1240 us), the fp32 backward, whose
// column fragments are single floats, loses 4% or more, and the dQ kernel gains nothing.
#pragma once

#include "ssa_common.h"

namespace ssa {
namespace tile {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

enum Swizzle { kNarrow = 0, kWide = 1 };  // (see the head of the file)

template <int RB, int SW>
__device__ __forceinline__ int swz(int r) {
  if constexpr (SW == kNarrow) return ((r & 3) << 1) | ((r >> 2) & 1);
  if constexpr (RB >= 256) return ((r & 3) << 2) | ((r >> 2) & 3);
  return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of RB bytes.
template <int RB, int SW = kNarrow>
__device__ __forceinline__ int chunk_at(int r, int c) {
  return r * RB + ((c ^ swz<RB, SW>(r)) << 4);
}

template <typename T>
struct Op;

// bf16 storage: one 32x32x16 product per fragment.
template <>
struct Op<uint16_t> {
  static constexpr int kEsize = 2;
  struct Frag {
    uint4 v;
  };
  static __device__ __forceinline__ f32x16 mfma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c,
                                                   0, 0, 0);
  }
  static __device__ __forceinline__ Frag zero() { return Frag{make_uint4(0u, 0u, 0u, 0u)}; }
  // Eight consecutive elements in global memory (16-byte aligned).
  static __device__ __forceinline__ Frag load(const uint16_t* p) { return Frag{*reinterpret_cast<const uint4*>(p)}; }
  // Columns 16c + 8 (l / 32) .. + 7 of tile row row0 + l % 32.
  template <int RB, int SW = kNarrow>
  static __device__ __forceinline__ Frag row_frag(const char* t, int row0, int c, int lane) {
    const int r = row0 + (lane & 31);
    return Frag{*reinterpret_cast<const uint4*>(t + chunk_at<RB, SW>(r, 2 * c + (lane >> 5)))};
  }
  // Column d0 + l % 32 of rows row0 + 4 (l / 32) + {0..3, 8..11} (row0 a multiple of 16).
  template <int RB, int SW = kNarrow>
  static __device__ __forceinline__ Frag col_frag(const char* t, int row0, int d0, int lane) {
    const int i = lane & 15;
    const int r = row0 + 4 * (lane >> 5) + (i >> 2);
    const int ch = (d0 >> 3) + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
    const char* p = t + (i & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + chunk_at<RB, SW>(r, ch)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + chunk_at<RB, SW>(r + 8, ch)));
    const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
    return Frag{make_uint4(a.x, a.y, b.x, b.y)};
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    // v_cvt_pk_bf16_f32, round to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
  // Registers 8c .. 8c + 7 of a score tile as a B operand.  Weights and score
  // gradients round to bf16 here, once (the products' inputs are bf16; the sums
  // stay fp32).
  static __device__ __forceinline__ Frag pack(const f32x16& s, int c) {
    return Frag{make_uint4(pack2(s[8 * c], s[8 * c + 1]), pack2(s[8 * c + 2], s[8 * c + 3]),
                           pack2(s[8 * c + 4], s[8 * c + 5]), pack2(s[8 * c + 6], s[8 * c + 7]))};
  }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float s) {
    const uint32_t x[4] = {a.v.x, a.v.y, a.v.z, a.v.w}, y[4] = {b.v.x, b.v.y, b.v.z, b.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
      s = fmaf(__uint_as_float(x[i] & 0xFFFF0000u), __uint_as_float(y[i] & 0xFFFF0000u), s);
    }
    return s;
  }
  // Four consecutive outputs, rounded once.
  static __device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(a, b), pack2(c, d));
  }
  static __device__ __forceinline__ void store1(uint16_t* p, float a) { *p = f32_to_bf16_rne(a); }
  // What rounding leaves.
  static __device__ __forceinline__ float left(float a) { return a - __uint_as_float(pack2(a, 0.0f) << 16); }
};

// fp32 storage: the same fragments as eight 32x32x2 products.
template <>
struct Op<float> {
  static constexpr int kEsize = 4;
  struct Frag {
    float v[8];
  };
  static __device__ __forceinline__ f32x16 mfma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag zero() { return Frag{{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}}; }
  static __device__ __forceinline__ Frag of(float4 a, float4 b) { return Frag{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
  static __device__ __forceinline__ Frag load(const float* p) {
    return of(*reinterpret_cast<const float4*>(p), *reinterpret_cast<const float4*>(p + 4));
  }
  template <int RB, int SW = kNarrow>
  static __device__ __forceinline__ Frag row_frag(const char* t, int row0, int c, int lane) {
    const int r = row0 + (lane & 31), ch = 4 * c + 2 * (lane >> 5);
    return of(*reinterpret_cast<const float4*>(t + chunk_at<RB, SW>(r, ch)),
              *reinterpret_cast<const float4*>(t + chunk_at<RB, SW>(r, ch + 1)));
  }
  template <int RB, int SW = kNarrow>
  static __device__ __forceinline__ Frag col_frag(const char* t, int row0, int d0, int lane) {
    const int d = d0 + (lane & 31);
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = row0 + 4 * (lane >> 5) + (i & 3) + 8 * (i >> 2);
      f.v[i] = *reinterpret_cast<const float*>(t + chunk_at<RB, SW>(r, d >> 2) + (d & 3) * 4);
    }
    return f;
  }
  static __device__ __forceinline__ Frag pack(const f32x16& s, int c) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = s[8 * c + i];
    return f;
  }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(a.v[i], b.v[i], s);
    return s;
  }
  static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
  static __device__ __forceinline__ void store1(float* p, float a) { *p = a; }
  static __device__ __forceinline__ float left(float) { return 0.0f; }
};

// Rows read through a buffer resource whose base moves with the tile: the address of
// a load is one 32-bit offset a thread keeps, and chunks and rows that do not exist
// (offsets past `bytes`) read as zeros with no branch.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kNoChunk = 0x80000000u;     // an offset past any resource
constexpr int kAllBytes = 0x7FFFFFF0;          // a resource whose rows all exist
constexpr int64_t kMostRowBytes = 1 << 24;     // of a row stride: the offsets of a tile's 128 rows stay below kAllBytes

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* base, int bytes) {
  // (word 3: raw 32-bit data)
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
__device__ __forceinline__ uint4 row_load(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(offset), 0, 0);
  return make_uint4(x.x, x.y, x.z, x.w);
}

// Waits for fragments loaded before a loop.  A load still out at the loop's head makes
// the compiler wait for every load at its first use in the body, the next tile's that
// were just issued among them.
__device__ __forceinline__ void settle(uint32_t& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void settle(float& x) { asm volatile("" : "+v"(x)); }
template <int N>
__device__ __forceinline__ void settle(Op<uint16_t>::Frag (&f)[N]) {
#pragma unroll
  for (int c = 0; c < N; ++c) {
    settle(f[c].v.x);
    settle(f[c].v.y);
    settle(f[c].v.z);
    settle(f[c].v.w);
  }
}
template <int N>
__device__ __forceinline__ void settle(Op<float>::Frag (&f)[N]) {
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) settle(f[c].v[i]);
}

// Keeps what uses x inside the wave-uniform branch it stands in.  Left alone, the
// compiler runs the mask's compares and selects for every tile (three instructions
// a score beside the eight that a score takes) rather than jump over them where a
// tile is seen whole.
__device__ __forceinline__ int in_branch(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The other half-wave's value of a lane's column.
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// Reductions over the 64 lanes of a wave (all lanes active) to a scalar, in six DPP
// steps: row_shr 1, 2, 4, 8 fold each 16-lane row into its last lane, row_bcast 15
// and 31 fold the rows into lane 63.  A lane whose source does not exist takes its
// own value.  (A ladder of shuffles costs an LDS round trip a step: four reductions
// of one took a microsecond at the head of every block.)
template <typename F>
__device__ __forceinline__ int wave_fold(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int wave_min_i(int x) {
  return wave_fold(x, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ int wave_max_i(int x) {
  return wave_fold(x, [](int a, int b) { return max(a, b); });
}
__device__ __forceinline__ float wave_max(float x) {
  return __int_as_float(wave_fold(__float_as_int(x), [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  }));
}
// (a sum counts each lane once: lanes without a source add 0)
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// The score rule, in log2 units (weights are exp2 of differences):
//   no cap:  x = (q.k) c1 - slope |pos - j|,          c1 = log2(e) / scale
//   cap c:   x = c2 tanh((q.k) c1) - slope |pos - j|,  c1 = 1 / (scale c), c2 = c log2(e)
// slope already carries log2(e).
struct ScoreRule {
  float c1, c2;
  int cap;              // scores go through the tanh: kDirect or kSeries of bf16's
  const float* slopes;  // null, or [h_q]
};
enum CapKind { kNoCap = 0, kDirect = 1, kSeries = 2 };

// tanh for the bf16 kernels.  kDirect: 1 - 2 / (exp(2y) + 1), off by 2^-22 (v_exp_f32 and
// v_rcp_f32 are good to an ulp), which puts a score and its weight off by c 2^-22: up to
// kMostDirectCap no more than 2^-12, a sixteenth of what rounding the weight to bf16 may
// leave.  kSeries, for larger caps, is good to a relative 2^-20, so that c tanh(s / c)
// keeps s however large c is: below 1/4 the series to y^7 (the first term left out is
// 62 / 2835 y^9), from there on the same as kDirect (8192 causal rows, 32 / 8 heads, d = 64,
// caps of 1025 and 1024: 745 us against 545, backward 2180 against 1610).  The fp32 kernels
// take the library's.
constexpr float kMostDirectCap = 1024.0f;

template <typename T, int CAP>
__device__ __forceinline__ float cap_tanh(float y) {
  if constexpr (sizeof(T) == 4) return tanhf(y);
  const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
  const float t = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  if constexpr (CAP == kDirect) return t;
  const float w = y * y, u = fmaf(w, fmaf(w, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f);
  return fabsf(y) < 0.25f ? fmaf(y * w, u, y) : t;
}

// The slope of a query head in log2 units (0: none).
__device__ __forceinline__ float slope_of(const ScoreRule& r, int hq) {
  return r.slopes != nullptr ? r.slopes[hq] * kLog2e : 0.0f;
}

// What the kernels keep of a product until its weight: z with x = a z + b, a and b
// the same for every score of the call, so that the running maximum, the
// subtraction of the reference and b cost one fma in the exponent.
//   kPlain  z = q.k
//   kCap    bf16: z = 1 / (exp(2y) + 1), of which tanh y = 1 - 2 z and
//           1 - tanh^2 = 4 (z - z^2); larger scores have smaller z.  fp32: z = tanh y
//   kBias   z = x (a distance bias, with or without a cap)
//   kFar    bf16: z = x, with a cap past kMostDirectCap and with or without a bias
enum RuleKind { kPlain = 0, kCap = 1, kBias = 2, kFar = 3 };

constexpr bool has_bias(int kind) { return kind == kBias || kind == kFar; }

template <typename T, int KIND>
struct Rule {
  static constexpr bool kDown = KIND == kCap && sizeof(T) == 2;
  static constexpr float kHidden = kDown ? INFINITY : -INFINITY;  // z of x = -inf
  // the gradient's factor 1 - tanh^2 is slope() times this
  static constexpr float kSlopeUnit = kDown ? 4.0f : 1.0f;
  float c, a, b;

  __device__ __forceinline__ explicit Rule(const ScoreRule& r) {
    c = kDown ? r.c1 * (2.0f * kLog2e) : r.c1;
    a = KIND == kPlain ? r.c1 : (kDown ? -2.0f * r.c2 : (KIND == kCap ? r.c2 : 1.0f));
    b = kDown ? r.c2 : 0.0f;
  }
  // dist: |position - key| or its negative (kBias, kFar)
  __device__ __forceinline__ float z(const ScoreRule& r, float dot, float slope, float dist) const {
    if constexpr (KIND == kPlain) return dot;
    if constexpr (kDown) return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * c) + 1.0f);
    if constexpr (KIND == kCap) return tanhf(dot * c);
    float x = dot * c;
    if constexpr (KIND == kFar)
      x = r.c2 * cap_tanh<T, kSeries>(x);
    else if (r.cap)
      x = r.c2 * cap_tanh<T, kDirect>(x);
    return fmaf(-slope, fabsf(dist), x);
  }
  // z, and the gradient's factor over kSlopeUnit
  __device__ __forceinline__ float z(const ScoreRule& r, float dot, float slope, float dist, float& f) const {
    f = 1.0f;
    if constexpr (has_bias(KIND)) {
      float x = dot * c;
      if (KIND == kFar || r.cap) {
        const float t = cap_tanh<T, KIND == kFar ? kSeries : kDirect>(x);
        f = fmaf(-t, t, 1.0f);
        x = r.c2 * t;
      }
      return fmaf(-slope, fabsf(dist), x);
    }
    const float v = z(r, dot, slope, dist);
    if constexpr (kDown) f = fmaf(-v, v, v);
    if constexpr (KIND == kCap && !kDown) f = fmaf(-v, v, 1.0f);
    return v;
  }
  static __device__ __forceinline__ float better(float x, float y) { return kDown ? fminf(x, y) : fmaxf(x, y); }
};

template <typename T>
RuleKind rule_kind(const ScoreRule& r) {
  if (sizeof(T) == 2 && r.cap == kSeries) return kFar;
  return r.slopes != nullptr ? kBias : (r.cap ? kCap : kPlain);
}

// exp2 of a difference of scores: the instruction's (an ulp; a result below
// 2^-126 is 0, a weight that no fp32 sum of weights up to 1 can hold).
__device__ __forceinline__ float exp2_w(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace tile
}  // namespace ssa
