// Rotary positions with several axes (ssa_rope_axes): q and k of images and video,
// whose tokens have a position on each of up to four axes (time, height, width).
//
// The rot / 2 feature pairs (m, m + rot / 2) are shared out among the axes in
// sections; pair m of axis a turns by ang = pos[a][b][i] freq[m]:
//   y[m]           = x[m] cos ang - x[m + rot / 2] sin ang
//   y[m + rot / 2] = x[m + rot / 2] cos ang + x[m] sin ang
// and features from rot on pass through.
//
// The angle is formed and reduced to an eighth of a turn in 64 bits, where far
// positions would lose it in 32, and its sine and cosine are Taylor polynomials
// in fp32 (the argument is at most pi / 4, the first term left out below 2e-9).
// A block takes a few tokens: their angles first, one a thread, into LDS, then all
// their heads of q and k, 16 bytes of each half of the pairs a thread, neighbouring
// threads on neighbouring chunks.  The 64-bit work is done once for the heads and
// the rest is bound by reading and writing q and k: 32768 tokens, 32 / 8 heads, d = 128,
// bf16 132 us, 5.1 TB/s (a large copy reads and writes 4.95).

#include "ssa_tile.h"

namespace ssa {
namespace {

constexpr int kAxThreads = 256;

struct AxesParams {
  const void *q, *k, *pos;
  void *q_out, *k_out;
  const double* freqs;
  int64_t n, rows;  // rows = batch * n
  int h_q, h_k, d, half, rot, items, tokens;  // items: chunks of a head; tokens: of a block
  int cut1, cut2, cut3;                            // first pairs of axes 1, 2, 3
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, qo_sb, qo_sn, qo_sh, ko_sb, ko_sn, ko_sh, p_sa, p_sb;
  float sign;  // -1: the transpose
};

// cos and sin of 2 pi rev.
__device__ __forceinline__ void turn(double rev, float& c, float& s) {
  const double y = rev * 4.0;
  const double k = __builtin_rint(y);
  const float a = static_cast<float>((y - k) * 1.57079632679489661923);
  const int quad = static_cast<int>(static_cast<int64_t>(k) & 3);
  const float z = a * a;
  float sn = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  sn = fmaf(z, sn, 8.33333333e-3f);
  sn = fmaf(z, sn, -1.66666667e-1f);
  sn = fmaf(a * z, sn, a);
  float cs = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  cs = fmaf(z, cs, -1.38888889e-3f);
  cs = fmaf(z, cs, 4.16666667e-2f);
  cs = fmaf(z, cs, -0.5f);
  cs = fmaf(z, cs, 1.0f);
  const float u = quad & 1 ? sn : cs, w = quad & 1 ? cs : sn;
  c = (quad == 1 || quad == 2) ? -u : u;
  s = quad >= 2 ? -w : w;
}

template <typename T, int VEC>
struct Chunk {
  float v[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      v[0] = ld(p);
    } else if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC == 1) {
      tile::Op<T>::store1(p, v[0]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      using O = tile::Op<uint16_t>;
      *reinterpret_cast<uint4*>(p) = make_uint4(O::pack2(v[0], v[1]), O::pack2(v[2], v[3]), O::pack2(v[4], v[5]), O::pack2(v[6], v[7]));
    }
  }
};

constexpr int kAxUnroll = 4;  // chunks of a thread whose loads are in flight together

template <typename T, typename P, int VEC>
__global__ __launch_bounds__(kAxThreads) void rope_axes_kernel(AxesParams p) {
  extern __shared__ __align__(16) float lds[];  // [tokens][half] cosines, then sines
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.rows - row0));
  float *cs = lds, *sn = lds + p.tokens * p.half;
  for (int x = threadIdx.x; x < tokens * p.half; x += kAxThreads) {
    const int tk = x / p.half, m = x - tk * p.half;
    const int64_t row = row0 + tk, b = row / p.n, i = row - b * p.n;
    const int axis = (m >= p.cut1) + (m >= p.cut2) + (m >= p.cut3);
    const double ang = static_cast<double>(static_cast<const P*>(p.pos)[axis * p.p_sa + b * p.p_sb + i]) * p.freqs[m];
    float c, s;
    turn(ang * 0.15915494309189533577, c, s);
    cs[x] = c;
    sn[x] = s * p.sign;
  }
  const int pairs = p.half / VEC, heads = p.h_q + p.h_k, all = tokens * heads * p.items;
  __syncthreads();
  for (int e0 = threadIdx.x; e0 < all; e0 += kAxThreads * kAxUnroll) {
    const T* src[kAxUnroll];
    T* dst[kAxUnroll];
    int at[kAxUnroll];  // the chunk's first angle, -1 where it passes through
    Chunk<T, VEC> x1[kAxUnroll], x2[kAxUnroll];
#pragma unroll
    for (int u = 0; u < kAxUnroll; ++u) {
      const uint32_t e = min(e0 + u * kAxThreads, all - 1);
      const uint32_t w = e / static_cast<uint32_t>(p.items);
      const int item = static_cast<int>(e - w * p.items);
      const uint32_t tk = w / static_cast<uint32_t>(heads);
      const int h = static_cast<int>(w - tk * heads);
      int64_t b = 0, i = row0 + tk;
      if (i >= p.n) {
        b = i / p.n;
        i -= b * p.n;
      }
      const bool isq = h < p.h_q;
      src[u] = isq ? static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_sn + h * p.q_sh
                   : static_cast<const T*>(p.k) + b * p.k_sb + i * p.k_sn + (h - p.h_q) * p.k_sh;
      dst[u] = isq ? static_cast<T*>(p.q_out) + b * p.qo_sb + i * p.qo_sn + h * p.qo_sh
                   : static_cast<T*>(p.k_out) + b * p.ko_sb + i * p.ko_sn + (h - p.h_q) * p.ko_sh;
      const int j = item < pairs ? item * VEC : p.rot + (item - pairs) * VEC;
      at[u] = item < pairs ? static_cast<int>(tk) * p.half + j : -1;
      src[u] += j;
      dst[u] += j;
      x1[u].load(src[u]);
      if (at[u] >= 0) x2[u].load(src[u] + p.half);
    }
#pragma unroll
    for (int u = 0; u < kAxUnroll; ++u) {
      if (e0 + u * kAxThreads >= all) break;
      if (at[u] < 0) {
        x1[u].store(dst[u]);
        continue;
      }
      Chunk<T, VEC> y1, y2;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float c = cs[at[u] + v], s = sn[at[u] + v];
        y1.v[v] = fmaf(x1[u].v[v], c, -(x2[u].v[v] * s));
        y2.v[v] = fmaf(x2[u].v[v], c, x1[u].v[v] * s);
      }
      y1.store(dst[u]);
      y2.store(dst[u] + p.half);
    }
  }
}

template <typename T, typename P>
int launch_axes(AxesParams& p, bool wide, hipStream_t st) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int vec = wide ? V : 1;
  p.items = (p.half + p.d - p.rot) / vec;
  // A token or more of angles for every thread of a block, fewer where that leaves
  // fewer than four blocks a CU.
  int64_t tokens = kAxThreads / p.half;
  if (tokens > p.rows / 1024) tokens = p.rows / 1024;
  p.tokens = static_cast<int>(tokens > 1 ? tokens : 1);
  const int64_t grid = ceil_div(p.rows, p.tokens);
  if (grid > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "ssa_rope_axes: too many rows");
  const size_t bytes = static_cast<size_t>(2) * p.tokens * p.half * sizeof(float);
  const void* kernel = wide ? reinterpret_cast<const void*>(rope_axes_kernel<T, P, V>) : reinterpret_cast<const void*>(rope_axes_kernel<T, P, 1>);
  if (int rc = reserve_lds(kernel, bytes, "ssa_rope_axes")) return rc;
  if (wide)
    rope_axes_kernel<T, P, V><<<dim3(static_cast<unsigned>(grid)), dim3(kAxThreads), bytes, st>>>(p);
  else
    rope_axes_kernel<T, P, 1><<<dim3(static_cast<unsigned>(grid)), dim3(kAxThreads), bytes, st>>>(p);
  return check_launch("ssa_rope_axes");
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" int ssa_rope_axes(const void* q, const void* k, int dtype, int64_t batch, int64_t n, int h_q, int h_k, int d,
                             int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                             const void* positions, int pos_dtype, int64_t p_sa, int64_t p_sb, int axes,
                             const int32_t* sections, const double* freqs, int rot, int inverse, void* q_out, int64_t qo_sb,
                             int64_t qo_sn, int64_t qo_sh, void* k_out, int64_t ko_sb, int64_t ko_sn, int64_t ko_sh,
                             void* stream) {
  const char* fn = "ssa_rope_axes";
  if (dtype != SSA_DTYPE_F32 && dtype != SSA_DTYPE_BF16) return fail(SSA_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", fn);
  if (pos_dtype != SSA_INDEX_I32 && pos_dtype != SSA_INDEX_I64)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: positions must be int32 or int64", fn);
  if (batch < 0 || n < 0 || h_q <= 0 || h_k < 0 || d <= 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape batch=%lld n=%lld h_q=%d h_k=%d d=%d", fn, (long long)batch,
                (long long)n, h_q, h_k, d);
  if (rot <= 0 || rot > d || (rot & 1))
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: rot=%d must be even and in (0, d=%d]", fn, rot, d);
  if (h_q > 4096 || h_k > 4096 || d > 4096)
    return fail(SSA_ERR_UNSUPPORTED, "%s: heads and head_dim must be at most 4096", fn);
  if (axes < 1 || axes > 4) return fail(SSA_ERR_UNSUPPORTED, "%s: axes=%d must be in [1, 4]", fn, axes);
  if (!sections) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  int64_t sum = 0;
  int cut[4] = {rot, rot, rot, rot};  // (past the last pair: axes that do not exist hold none)
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 0) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: section %d is negative", fn, a);
    if (a > 0) cut[a - 1] = static_cast<int>(sum);
    sum += sections[a];
    if (sum > rot) break;
  }
  if (sum != rot / 2)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: the sections must hold the rot / 2 = %d pairs", fn, rot / 2);
  if (batch == 0 || n == 0) return SSA_OK;
  if (!q || !q_out || (h_k > 0 && (!k || !k_out)) || !positions || !freqs)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  AxesParams p{};
  p.q = q; p.k = k; p.pos = positions; p.q_out = q_out; p.k_out = k_out; p.freqs = freqs;
  p.n = n; p.rows = batch * n; p.h_q = h_q; p.h_k = h_k; p.d = d; p.half = rot / 2; p.rot = rot;
  p.cut1 = cut[0]; p.cut2 = cut[1]; p.cut3 = cut[2];
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh; p.k_sb = k_sb; p.k_sn = k_sn; p.k_sh = k_sh;
  p.qo_sb = qo_sb; p.qo_sn = qo_sn; p.qo_sh = qo_sh; p.ko_sb = ko_sb; p.ko_sn = ko_sn; p.ko_sh = ko_sh;
  p.p_sa = p_sa; p.p_sb = p_sb;
  p.sign = inverse ? -1.0f : 1.0f;
  // 16-byte chunks where every row and both halves of the pairs allow them
  const int e = dtype == SSA_DTYPE_F32 ? 4 : 2, v = 16 / e;
  auto al = [&](const void* x, int64_t sb, int64_t sn, int64_t sh) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && sb % v == 0 && sn % v == 0 && sh % v == 0;
  };
  const bool wide = p.half % v == 0 && (d - rot) % v == 0 && al(q, q_sb, q_sn, q_sh) && al(q_out, qo_sb, qo_sn, qo_sh) &&
                    (h_k == 0 || (al(k, k_sb, k_sn, k_sh) && al(k_out, ko_sb, ko_sn, ko_sh)));
  hipStream_t st = as_stream(stream);
  if (dtype == SSA_DTYPE_F32)
    return pos_dtype == SSA_INDEX_I64 ? launch_axes<float, int64_t>(p, wide, st) : launch_axes<float, int32_t>(p, wide, st);
  return pos_dtype == SSA_INDEX_I64 ? launch_axes<uint16_t, int64_t>(p, wide, st) : launch_axes<uint16_t, int32_t>(p, wide, st);
}
