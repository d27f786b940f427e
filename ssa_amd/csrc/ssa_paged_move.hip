// Rows of a paged cache moved: read back to contiguous tensors (ssa_paged_read), and the kept
// path of a drafted tree to the front of its tokens (ssa_paged_keep).
//
// Both are copies, bound by memory where they are large and by a launch where they are not
// (reading back 32 tokens 5 us).

#include "ssa_dense_rows.h"
#include "ssa_internal.h"
#include "ssa_tile.h"

namespace ssa {
namespace {

using namespace tile;

struct Pool {
  void* at;
  float* scale;  // of 8-bit codes
  int64_t sp, st, sh, c_sp, c_st, c_sh;
};

struct MoveParams {
  Pool k, v;
  const int32_t *table, *starts, *first;  // read: rows of a sequence, its first key
  const int32_t *cached, *kept;           // keep
  int64_t table_stride, kept_stride, tokens;
  int batch, h_kv, d, max_pages, page_log2, num_pages, e4m3, most;
  void *k_out, *v_out;
  int32_t* error_flag;
};

__device__ __forceinline__ void flag(const MoveParams& p) {
  if (p.error_flag != nullptr) atomicOr(p.error_flag, 1);
}

// The page of key j of sequence b, -1 where there is none.
__device__ __forceinline__ int page_of(const MoveParams& p, int b, int64_t j) {
  if (j < 0 || j >= static_cast<int64_t>(p.max_pages) << p.page_log2) return -1;
  const int pg = p.table[b * p.table_stride + (j >> p.page_log2)];
  return static_cast<unsigned>(pg) < static_cast<unsigned>(p.num_pages) ? pg : -1;
}

// Eight codes * scale for results in bf16.  fp32's products are rounded again as the exact ones would be,
// unless one lies halfway between two of bf16 and is not exact itself (13 of 2 million): it moves to the side
// of the exact one, which fp64 holds (24 bits by 8).  2048 tokens of 8 heads: 6.7 us, 7.4 where fp64 forms every
// product, 6.2 rounded twice.
__device__ __forceinline__ void bf16_products(float f, const float (&c)[8], float (&o)[8]) {
  bool halfway = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    o[i] = f * c[i];
    halfway |= (__float_as_uint(o[i]) & 0xFFFFu) == 0x8000u;
  }
  if (!halfway) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(o[i]);
    const double x = static_cast<double>(f) * static_cast<double>(c[i]), y = static_cast<double>(o[i]);
    if ((u & 0xFFFFu) == 0x8000u && x != y && finite(o[i])) o[i] = __uint_as_float(fabs(y) < fabs(x) ? u + 1 : u - 1);
  }
}

// Eight features a thread.  T is the output's type, S the pages'.
template <typename T, typename S>
__global__ __launch_bounds__(256) void read_kernel(MoveParams p) {
  const int per = p.d / 8;
  const int64_t total = p.tokens * p.h_kv * per, t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= 2 * total) return;
  const bool isv = t >= total;
  const int64_t u = isv ? t - total : t, row = u / per;
  const int c = static_cast<int>(u - row * per) * 8;
  const int64_t tok = row / p.h_kv;
  const int h = static_cast<int>(row - tok * p.h_kv);
  int x = 0, y = p.batch + 1;  // the first start past the token
  while (x < y) {
    const int mid = (x + y) >> 1;
    if (p.starts[mid] <= tok)
      x = mid + 1;
    else
      y = mid;
  }
  const int b = x - 1;
  uint4 w[sizeof(T) / 2];
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 2; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
  if (b >= 0 && b < p.batch) {
    const int64_t j = p.first[b] + (tok - p.starts[b]);
    const int64_t pg = page_of(p, b, j), r = j & ((1 << p.page_log2) - 1);
    if (pg < 0) {
      flag(p);
    } else {
      const Pool& pool = isv ? p.v : p.k;
      const S* src = static_cast<const S*>(pool.at) + pg * pool.sp + r * pool.st + h * pool.sh + c;
      if constexpr (sizeof(S) == 1) {
        const float f = pool.scale[pg * pool.c_sp + r * pool.c_st + h * pool.c_sh];
        const uint2 code = *reinterpret_cast<const uint2*>(src);
        float o[8], x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = code_value(static_cast<uint8_t>((i < 4 ? code.x : code.y) >> (8 * (i & 3))), p.e4m3);
        if constexpr (sizeof(T) == 2) {
          bf16_products(f, x, o);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = f * x[i];
        }
        if constexpr (sizeof(T) == 2) {
          w[0] = make_uint4(Op<uint16_t>::pack2(o[0], o[1]), Op<uint16_t>::pack2(o[2], o[3]), Op<uint16_t>::pack2(o[4], o[5]),
                            Op<uint16_t>::pack2(o[6], o[7]));
        } else {
          w[0] = make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
          w[1] = make_uint4(__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7]));
        }
      } else {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(src)[i];
      }
    }
  }
  T* dst = static_cast<T*>(isv ? p.v_out : p.k_out) + row * p.d + c;
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(dst)[i] = w[i];
}

// Moves one piece (of type U) of every kept row of a sequence, sixteen rows' loads in flight.  Kept
// rows ascend, so that the t-th lies at or behind its place: what is written is never read later.
template <typename U>
__device__ __forceinline__ void keep_piece(int n, const int2* s_from, const int2* s_to, char* base, int64_t sp, int64_t st) {
  constexpr int kAtOnce = 16;
  for (int t0 = 0; t0 < n; t0 += kAtOnce) {
    U x[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int2 a = s_from[min(t0 + i, n - 1)];
      x[i] = *reinterpret_cast<const U*>(base + a.x * sp + a.y * st);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (t0 + i < n) {
        const int2 a = s_to[t0 + i];
        *reinterpret_cast<U*>(base + a.x * sp + a.y * st) = x[i];
      }
  }
}

constexpr int kMostKept = 64;

// A thread takes a piece of a head's rows of K or V, of all kept tokens; E bytes an element.  Blocks of
// one wave, which looks the rows up for itself: rows that are in their place already, or that have no page at one
// end, are left out.
template <int E>
__global__ __launch_bounds__(64) void keep_kernel(MoveParams p) {
  using U = std::conditional_t<E == 1, uint2, uint4>;
  __shared__ int2 s_from[kMostKept], s_to[kMostKept];  // page, row of it
  __shared__ int s_n;
  const int b = blockIdx.y;
  {  // the kept tokens up to the first one below 0, or the first that does not ascend
    const int lane = threadIdx.x, first = p.cached[b];
    const int x = lane < p.most ? p.kept[b * p.kept_stride + lane] : -1;
    const int before = __shfl_up(x, 1, 64);
    const uint64_t end = __ballot(x < 0), fall = __ballot(lane > 0 && x >= 0 && x <= before);
    const int n = end != 0 ? __builtin_ctzll(end) : 64, good = fall != 0 ? __builtin_ctzll(fall) : 64;
    bool on = first >= 0 && lane < min(n, good), bad = first < 0 || good < n;
    const int64_t from = static_cast<int64_t>(first) + x, to = static_cast<int64_t>(first) + lane;
    int pg = 0, pt = 0;
    if (on) {
      pg = page_of(p, b, from);
      pt = page_of(p, b, to);
      bad |= pg < 0 || pt < 0;
      on = pg >= 0 && pt >= 0 && x != lane;
    }
    const uint64_t go = __ballot(on);
    const int at = __popcll(go & ((uint64_t(1) << lane) - 1)), mask = (1 << p.page_log2) - 1;
    if (on) {
      s_from[at] = make_int2(pg, static_cast<int>(from & mask));
      s_to[at] = make_int2(pt, static_cast<int>(to & mask));
    }
    if (bad) flag(p);
    if (lane == 0) s_n = __popcll(go);
  }
  __syncthreads();
  const int n = s_n, per = p.d * E / static_cast<int>(sizeof(U)), rows = 2 * p.h_kv;
  const int at = blockIdx.x * 64 + threadIdx.x;
  if (n == 0) return;
  if (at < rows * per) {
    const int row = at / per, c = at - row * per;
    const bool isv = row >= p.h_kv;
    const Pool& pool = isv ? p.v : p.k;
    char* base = static_cast<char*>(pool.at) + (isv ? row - p.h_kv : row) * pool.sh * E + c * static_cast<int>(sizeof(U));
    keep_piece<U>(n, s_from, s_to, base, pool.sp * E, pool.st * E);
  } else if (E == 1 && at < rows * (per + 1)) {
    const int row = at - rows * per;
    const bool isv = row >= p.h_kv;
    const Pool& pool = isv ? p.v : p.k;
    keep_piece<uint32_t>(n, s_from, s_to, reinterpret_cast<char*>(pool.scale + (isv ? row - p.h_kv : row) * pool.c_sh),
                         pool.c_sp * 4, pool.c_st * 4);
  }
}

int check_pool(const char* fn, const char* name, int page_dtype, const void* at, int64_t sp, int64_t st, int64_t sh,
               const float* scale, int64_t c0, int64_t c1, int64_t c2) {
  const bool held = page_dtype == SSA_DTYPE_I8 || page_dtype == SSA_DTYPE_E4M3;
  const int64_t e = held ? 1 : (page_dtype == SSA_DTYPE_F32 ? 4 : 2), unit = held ? 8 : 16;
  if (at == nullptr || (held && scale == nullptr)) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (reinterpret_cast<uintptr_t>(at) % unit != 0 || sp * e % unit != 0 || st * e % unit != 0 || sh * e % unit != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s must have rows aligned to %d bytes", fn, name, (int)unit);
  if (sp < 0 || st < 0 || sh < 0 || c0 < 0 || c1 < 0 || c2 < 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: %s must have strides from 0", fn, name);
  return SSA_OK;
}

int check_sizes(const char* fn, int page_dtype, int64_t batch, int h_kv, int d, int64_t num_pages, int page_size, int max_pages) {
  if (page_dtype < SSA_DTYPE_F32 || page_dtype > SSA_DTYPE_E4M3)
    return fail(SSA_ERR_UNSUPPORTED, "%s: pages hold f32, bf16, int8 or e4m3", fn);
  if (batch < 0 || h_kv <= 0 || d <= 0 || num_pages < 0 || max_pages < 0)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape batch=%lld h_kv=%d d=%d num_pages=%lld", fn, (long long)batch, h_kv, d,
                (long long)num_pages);
  if (d % 8 != 0 || d > 128) return fail(SSA_ERR_UNSUPPORTED, "%s: head_dim %d must be a multiple of 8, at most 128", fn, d);
  if (page_size < 8 || page_size > 4096 || (page_size & (page_size - 1)) != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: page_size %d must be a power of 2 in [8, 4096]", fn, page_size);
  if (batch > 0x7FFFFF || h_kv > 65536 || num_pages > 0x7FFFFFFF || static_cast<int64_t>(max_pages) * page_size > 0x7FFFFF00)
    return fail(SSA_ERR_UNSUPPORTED, "%s: sequences must be shorter than 2^31", fn);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" int ssa_paged_read(const void* k_pages, const void* v_pages, int page_dtype, const float* k_scales,
                              const float* v_scales, int64_t num_pages, int page_size, int h_kv, int d, int64_t kp_sp,
                              int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh, int64_t ks_sp,
                              int64_t ks_st, int64_t ks_sh, int64_t vs_sp, int64_t vs_st, int64_t vs_sh, int64_t batch,
                              const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                              const int32_t* first, int64_t tokens, int out_dtype, void* k_out, void* v_out,
                              int32_t* error_flag, void* stream) {
  const char* fn = "ssa_paged_read";
  if (int rc = check_sizes(fn, page_dtype, batch, h_kv, d, num_pages, page_size, max_pages)) return rc;
  const bool held = page_dtype == SSA_DTYPE_I8 || page_dtype == SSA_DTYPE_E4M3;
  if ((out_dtype != SSA_DTYPE_F32 && out_dtype != SSA_DTYPE_BF16) || (!held && out_dtype != page_dtype))
    return fail(SSA_ERR_UNSUPPORTED, "%s: rows are read as the pages' type, of 8 bits as f32 or bf16", fn);
  if (tokens < 0 || tokens > 0x7FFFFF00)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape tokens=%lld", fn, (long long)tokens);
  if (tokens == 0) return SSA_OK;
  if (batch < 1 || num_pages < 1 || max_pages < 1)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: batch, num_pages and max_pages must be positive", fn);
  if (!table || !starts || !first || !k_out || !v_out) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (int rc = check_pool(fn, "k_pages", page_dtype, k_pages, kp_sp, kp_st, kp_sh, k_scales, ks_sp, ks_st, ks_sh)) return rc;
  if (int rc = check_pool(fn, "v_pages", page_dtype, v_pages, vp_sp, vp_st, vp_sh, v_scales, vs_sp, vs_st, vs_sh)) return rc;
  if (reinterpret_cast<uintptr_t>(k_out) % 16 != 0 || reinterpret_cast<uintptr_t>(v_out) % 16 != 0)
    return fail(SSA_ERR_UNSUPPORTED, "%s: the outputs must be aligned to 16 bytes", fn);
  MoveParams p{};
  p.k = Pool{const_cast<void*>(k_pages), const_cast<float*>(k_scales), kp_sp, kp_st, kp_sh, ks_sp, ks_st, ks_sh};
  p.v = Pool{const_cast<void*>(v_pages), const_cast<float*>(v_scales), vp_sp, vp_st, vp_sh, vs_sp, vs_st, vs_sh};
  p.table = table; p.starts = starts; p.first = first;
  p.table_stride = table_stride; p.tokens = tokens;
  p.batch = static_cast<int>(batch); p.h_kv = h_kv; p.d = d;
  p.max_pages = max_pages; p.num_pages = static_cast<int>(num_pages);
  while ((1 << p.page_log2) < page_size) ++p.page_log2;
  p.e4m3 = page_dtype == SSA_DTYPE_E4M3;
  p.k_out = k_out; p.v_out = v_out; p.error_flag = error_flag;
  const int64_t blocks = ceil_div(2 * tokens * h_kv * (d / 8), 256);
  if (blocks > 0x7FFFFFFF) return fail(SSA_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  const dim3 grid(static_cast<unsigned>(blocks));
  hipStream_t st = as_stream(stream);
  const bool f32 = out_dtype == SSA_DTYPE_F32;
  if (held) {
    if (f32)
      read_kernel<float, uint8_t><<<grid, dim3(256), 0, st>>>(p);
    else
      read_kernel<uint16_t, uint8_t><<<grid, dim3(256), 0, st>>>(p);
  } else if (f32) {
    read_kernel<float, float><<<grid, dim3(256), 0, st>>>(p);
  } else {
    read_kernel<uint16_t, uint16_t><<<grid, dim3(256), 0, st>>>(p);
  }
  return check_launch(fn);
}

extern "C" int ssa_paged_keep(void* k_pages, void* v_pages, int page_dtype, float* k_scales, float* v_scales,
                              int64_t num_pages, int page_size, int h_kv, int d, int64_t kp_sp, int64_t kp_st, int64_t kp_sh,
                              int64_t vp_sp, int64_t vp_st, int64_t vp_sh, int64_t ks_sp, int64_t ks_st, int64_t ks_sh,
                              int64_t vs_sp, int64_t vs_st, int64_t vs_sh, int64_t batch, const int32_t* table,
                              int64_t table_stride, int max_pages, const int32_t* cached, const int32_t* kept,
                              int64_t kept_stride, int most_kept, int32_t* error_flag, void* stream) {
  const char* fn = "ssa_paged_keep";
  if (int rc = check_sizes(fn, page_dtype, batch, h_kv, d, num_pages, page_size, max_pages)) return rc;
  if (most_kept < 0) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: bad shape most_kept=%d", fn, most_kept);
  if (most_kept > kMostKept)
    return fail(SSA_ERR_UNSUPPORTED, "%s: at most %d tokens of a sequence are kept, not %d", fn, kMostKept, most_kept);
  if (batch == 0 || most_kept == 0) return SSA_OK;
  if (num_pages < 1 || max_pages < 1)
    return fail(SSA_ERR_INVALID_ARGUMENT, "%s: num_pages and max_pages must be positive", fn);
  if (!table || !cached || !kept) return fail(SSA_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (int rc = check_pool(fn, "k_pages", page_dtype, k_pages, kp_sp, kp_st, kp_sh, k_scales, ks_sp, ks_st, ks_sh)) return rc;
  if (int rc = check_pool(fn, "v_pages", page_dtype, v_pages, vp_sp, vp_st, vp_sh, v_scales, vs_sp, vs_st, vs_sh)) return rc;
  MoveParams p{};
  p.k = Pool{k_pages, k_scales, kp_sp, kp_st, kp_sh, ks_sp, ks_st, ks_sh};
  p.v = Pool{v_pages, v_scales, vp_sp, vp_st, vp_sh, vs_sp, vs_st, vs_sh};
  p.table = table; p.cached = cached; p.kept = kept;
  p.table_stride = table_stride; p.kept_stride = kept_stride;
  p.batch = static_cast<int>(batch); p.h_kv = h_kv; p.d = d; p.most = most_kept;
  p.max_pages = max_pages; p.num_pages = static_cast<int>(num_pages);
  while ((1 << p.page_log2) < page_size) ++p.page_log2;
  p.error_flag = error_flag;
  const bool held = page_dtype == SSA_DTYPE_I8 || page_dtype == SSA_DTYPE_E4M3;
  const int64_t pieces = 2 * h_kv * static_cast<int64_t>(held ? d / 8 + 1 : d / (page_dtype == SSA_DTYPE_F32 ? 4 : 8));
  hipStream_t st = as_stream(stream);
  for (int64_t b0 = 0; b0 < batch; b0 += 65535) {  // (a grid's second axis)
    MoveParams part = p;
    part.table += b0 * table_stride;
    part.cached += b0;
    part.kept += b0 * kept_stride;
    const dim3 grid(static_cast<unsigned>(ceil_div(pieces, 64)), static_cast<unsigned>(batch - b0 < 65535 ? batch - b0 : 65535));
    if (held)
      keep_kernel<1><<<grid, dim3(64), 0, st>>>(part);
    else if (page_dtype == SSA_DTYPE_F32)
      keep_kernel<4><<<grid, dim3(64), 0, st>>>(part);
    else
      keep_kernel<2><<<grid, dim3(64), 0, st>>>(part);
    if (int rc = check_launch(fn)) return rc;
  }
  return SSA_OK;
}
