// How the dense attention calls are cut into blocks, and the workspaces that follow: rules on
// sizes and types alone, in plain C++, so that a host test can ask for a call's cut.  Those that
// the kernels follow too (SSA_BOTH) stand here for both.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "ssa_hip.h"

#ifdef __HIPCC__
#define SSA_BOTH __host__ __device__ inline __attribute__((always_inline))
#else
#define SSA_BOTH inline
#endif

namespace ssa {

constexpr int kFew = 32;  // rows of a few-row block of ssa_paged_step

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a dense forward of `rows` rows (tokens x heads of a group) of each of `heads`
// KV heads over `keys` keys is cut: waves that share 32 rows, and parts of the keys.
struct DenseSplit {
  int kw, parts;
};
inline DenseSplit dense_split(int64_t rows, int64_t heads, int64_t keys, int64_t n_q, bool f32, bool wide, bool paged) {
  // Blocks of 128 rows, one wave a row, from 512 blocks on (two a CU).  Where they are
  // fewer (us a call, both sides measured; of 120 calls of 700 to 5000 keys and 10 to
  // 500 blocks the rule's cut is 4% slower than the best of 27 in the mean):
  DenseSplit s{1, 1};
  const int64_t blocks = div_up(rows, 128) * heads;
  if (blocks <= 0 || blocks >= 512 || keys <= 32) return s;
  // Two or four waves share each 32 rows and take turns at the keys (2500 causal rows of
  // 8 / 2 heads, d = 64, 158 blocks: 40 with two, 32 with four; 1500 of 32 / 8, d = 128,
  // 376 blocks: 54 with one or two, 67 with four).  Four read the keys four times as
  // often as one; bf16 is bound by that over long ones (6000: twice as slow), fp32 never
  // (4096 causal rows of 8 / 2 heads, d = 64: 194 with two, 187 with four).
  const bool one_block = f32 && wide;  // a CU holds one block, of two waves a row at most
  const int64_t four = f32 ? 256 : 176;
  if (blocks < four && keys > 64 && (f32 || keys < 4096) && !one_block)
    s.kw = 4;
  else if (blocks < 400)
    s.kw = 2;
  // Parts of the keys, joined by a second launch.  They pay where the rows are few
  // beside the keys, which each row then sees nearly all of; in a square causal or
  // document mask most parts of a row are empty (1500 rows of 12 / 4 heads, d = 128:
  // 35 in one part, 45 in three).  Long keys take as many parts as about 512 blocks
  // allow, of 384 keys at least, and waves share rows only where those are few still
  // (1200 x 8 rows over 16384 keys: 289 in one part, 138 in six); not two parts below
  // 8192 keys, where the join costs more.  Shorter ones take parts only until the blocks
  // fill the CUs once, of at least 384 keys (fp32 192: 140 x 4 rows of 2 heads over 700
  // keys 30 and 24 in one and three parts; bf16 18.6 and 20.3).  Over pages, whose rows
  // follow what is cached and whose tiles wait for their pages as well, half as long
  // parts and twice as many pay (915 x 3 rows of 2 heads over 2470 keys: 68 in one part,
  // 51 in three; 500 x 7 rows twice of 4 heads over 6500: 188 in three, 165 in four).
  const bool chunk = paged || 2 * n_q <= keys;
  int64_t want = 1, can = 1;
  if (chunk && keys >= 4096) {
    want = paged ? div_up(640, blocks) : (512 + blocks / 4) / blocks;
    can = keys / 384;
    if (!paged && (want < can ? want : can) == 2 && keys < 8192) want = 1;
    const int64_t all = blocks * (want < can ? want : can);
    s.kw = all > blocks && all >= 384 ? 1 : (paged && all < 64 && !one_block ? 4 : 2);
  } else if (chunk || one_block) {
    const int64_t all = blocks * s.kw;
    want = ((paged ? 512 : 256) + all / 2) / all;
    can = keys / (f32 || paged ? 192 : 384);
  }
  const int64_t parts = want < can ? want : can;
  s.parts = parts > 1 ? static_cast<int>(parts) : 1;
  return s;
}

// How a backward is cut, and its workspace: the rows' stats, the groups' bounds, and
// the parts of dK and dV.
struct BwdCut {
  int kw, key_groups, splits, groups;
  size_t stats, bounds, part, bytes;
};

inline BwdCut bwd_cut(int dtype, int64_t batch, int64_t n, int64_t n_q, int h_q, int h_kv, int d) {
  BwdCut l{};
  const int64_t rows = n_q * (h_q / h_kv), heads = batch * h_kv;
  const bool f32 = dtype == SSA_DTYPE_F32, wide = d > 64;
  l.groups = static_cast<int>(div_up(rows, 32));
  // dQ: waves share rows where blocks of 128 are few, earlier than in the forward
  // (no maximum to agree on): 1500 x 8 rows of 4 x 2 heads, 752 blocks, take the
  // same with one wave a row and with two; 2048 x 7 of 4 heads, 448 blocks, 5% less
  // with two; 4096 of 4 heads at d = 64, 128 blocks, 9% less with four.
  const int64_t qblocks = div_up(rows, 128) * heads;
  l.kw = qblocks >= 1024 || n <= 32 ? 1 : (qblocks >= 192 || n <= 64 || (f32 && wide) ? 2 : 4);
  // dK, dV: blocks of 128 keys, their rows cut into parts until 512 blocks (two a CU
  // where they fit; 1024 of the smaller ones of bf16 at d = 64, of which four do) fill
  // the device, at least 128 rows a part, one more part where that fills the last
  // round better.  With fewer than 256 blocks even so, blocks of 64 or 32 keys, whose
  // waves share keys.  Parts cost a write and a read of dK and dV in fp32: 64 blocks
  // (2048 keys, 28 / 4 heads, d = 128) take 395, 330, 266 and 300 us in 3, 4, 8 and 16.
  const int64_t target = !f32 && !wide ? 1024 : 512;
  l.key_groups = 4;
  for (;; l.key_groups /= 2) {
    const int64_t blocks = div_up(n, 32 * l.key_groups) * heads;
    int64_t s = blocks > 0 ? div_up(target, blocks) : 1;
    auto idle = [&](int64_t x) { return static_cast<double>(div_up(blocks * x, 256) * 256) / (blocks * x); };
    if (s > 1 && blocks > 0 && idle(s + 1) < idle(s) - 0.1) ++s;
    const int64_t most = rows / 128;
    l.splits = static_cast<int>(s < most ? s : (most > 1 ? most : 1));
    if (blocks * l.splits >= 256 || l.key_groups <= (wide ? 2 : 1)) break;
  }
  l.stats = 0;
  l.bounds = static_cast<size_t>(batch) * h_q * n_q * 16;
  l.part = l.bounds + static_cast<size_t>(batch) * l.groups * 16;
  l.bytes = l.part;
  if (l.splits > 1) l.bytes += 2 * static_cast<size_t>(l.splits) * batch * n * h_kv * (wide ? 128 : 64) * sizeof(float);
  return l;
}

// The backward of rows that see two intervals: blocks of keys, how many of a head run at a time
// (slots), the parts that dkv_kernel's plan may cut blocks into (extra, and one more for each that
// it cuts), and the workspace.  Few blocks of keys are all cut alike, as those of one interval are,
// with no plan (1024 x 2 rows of 8 / 2 heads, fp32, d = 64: the plan's two kernels take 13 us of 163).
struct TwoCut {
  bool planned;
  int64_t key_blocks;
  int slots, extra, most;
  size_t counts, entries, cut, part, part_floats, bytes;
};

inline TwoCut two_cut(const BwdCut& l, int dtype, int64_t batch, int64_t n, int h_kv, int d) {
  TwoCut t{};
  const bool f32 = dtype == SSA_DTYPE_F32, wide = d > 64;
  const int64_t keys = 32 * l.key_groups;
  t.key_blocks = div_up(n, keys) * batch;
  // a CU holds one block of bf16 at 128 features (its K and V lie in the LDS), two of the others
  t.slots = static_cast<int>(div_up(!f32 && wide ? 256 : 512, h_kv));
  t.extra = 4 * t.slots;
  t.most = t.extra + 3 * t.slots;
  t.planned = 4 * t.key_blocks > t.slots;
  // (no more parts than each block of keys with one for every group of rows)
  const int64_t all = t.key_blocks * l.groups, parts = all < t.most ? all : t.most;
  t.counts = l.bounds + 2 * static_cast<size_t>(batch) * l.groups * 16;
  if (!t.planned) {
    t.part = t.counts;
    t.part_floats = l.splits > 1 ? static_cast<size_t>(l.splits) * batch * n * h_kv * (wide ? 128 : 64) : 0;
    t.bytes = t.part + 2 * t.part_floats * sizeof(float);
    return t;
  }
  t.entries = (t.counts + static_cast<size_t>(t.key_blocks) * 4 + 15) / 16 * 16;
  t.cut = t.entries + static_cast<size_t>(t.key_blocks + t.most) * 16;
  t.part = t.cut + static_cast<size_t>(2 * t.slots + 1) * 16;
  t.part_floats = static_cast<size_t>(parts) * h_kv * keys * (wide ? 128 : 64);
  t.bytes = t.part + 2 * t.part_floats * sizeof(float);
  return t;
}

// What plan_list_kernel makes of a call whose blocks of keys are seen by `h` tiles of rows each,
// `total` in all.  A block with more than `share` of them is big, and cut into parts of plan_part
// tiles; of the others, whole ones, plan_left of the last round are cut into parts of plan_left_part.
SSA_BOTH int64_t plan_share(int64_t total, int slots, int least) {
  const int64_t share = (total + slots - 1) / slots;
  return share > least ? share : least;
}
// big: tiles of the big blocks
SSA_BOTH int plan_part(int64_t big, int extra, int least, int64_t share) {
  int64_t p = (big + extra - 1) / extra;
  p = p > least ? p : least;
  return static_cast<int>(p > share / 10 ? p : share / 10);
}
// How many of the `one` blocks that are not big, the shortest, are cut so that they fill a last round
// (0: none).  Blocks are sorted up to kSorted of them.
constexpr int kSorted = 2048;
SSA_BOTH int plan_left(int blocks, int one, int slots) {
  const int left = one % slots;
  return blocks <= kSorted && one > slots && one < 4 * slots && 10 * left < 7 * slots ? left : 0;
}
// sum: tiles of those
SSA_BOTH int plan_left_part(int64_t sum, int slots, int least) {
  const int64_t p = (sum + slots - 1) / slots;
  return static_cast<int>(p > least ? p : least);
}
// Parts of a block of h tiles that is cut (one at least: nobody sees it, and its zeros go through a part).
SSA_BOTH int plan_parts(int h, int part) { return h > part ? (h + part - 1) / part : 1; }

// The tiles of kt keys that the rows of a block see, [a_lo, a_hi) and [b_lo, b_hi) between them:
// [x0, x0 + n1), then [y0, y0 + n - n1), ascending.
struct Tiles {
  int x0, n1, y0, n;
  SSA_BOTH int at(int t) const { return t < n1 ? x0 + t : y0 + t - n1; }
};
SSA_BOTH Tiles tiles_of(int a_lo, int a_hi, int b_lo, int b_hi, int kt) {
  int x0 = a_lo / kt, x1 = a_hi > a_lo ? (a_hi - 1) / kt + 1 : x0;
  int y0 = b_lo / kt, y1 = b_hi > b_lo ? (b_hi - 1) / kt + 1 : y0;
  if (x1 == x0) {  // (one range)
    x0 = y0;
    x1 = y1;
    y1 = y0;
  }
  if (y1 > y0 && y0 < x0) {
    const int s0 = x0, s1 = x1;
    x0 = y0;
    x1 = y1;
    y0 = s0;
    y1 = s1;
  }
  if (y1 > y0 && y0 <= x1) {
    x1 = x1 > y1 ? x1 : y1;
    y1 = y0;
  }
  return Tiles{x0, x1 - x0, y0, x1 - x0 + y1 - y0};
}
// Those of a sequence's new tokens, at positions cached to len - 1, behind a window (0: none) with
// first keys.
SSA_BOTH Tiles seen_tiles(int cached, int len, int window, int sinks, int kt) {
  const int lo = window > 0 && cached + 1 - window > 0 ? cached + 1 - window : 0;
  const int far = window > 0 && len - window > 0 ? len - window : 0;
  return tiles_of(0, sinks < far ? sinks : far, lo, len, kt);
}

// The most keys of a sequence of max_len that its call reads: with a window, the first keys
// and those of the window and the new tokens, in whole tiles of up to 128.
inline int64_t seen_len(int64_t max_len, int64_t max_new, int64_t window, int64_t sinks) {
  if (window <= 0 || window >= max_len || sinks >= max_len) return max_len;
  const int64_t some = div_up(sinks, 128) * 128 + window + max_new + 256;
  return some < max_len ? some : max_len;
}

// Whether a call over pages of 8 bits is one for few_codes: bf16 queries, rows of whole 16-byte pieces
// where a lane loads 16, at most 16 rows a sequence, and of those at most two new tokens, which it adds one
// by one.  us a call (repeated on the same pages) by few_rows and few_codes, int8, d = 128, 4 KV heads of 4
// query heads, of 1 where 8 tokens are new:
//   new tokens                 1              2             4             8
//   32 sequences of 4000       51.4, 45.2     52.5, 46.0    54.3, 55.4    55.3, 57.3
//   32 of 200                  12.8, 12.2     13.0, 12.3    13.8, 15.4    13.1, 20.6
//   one of 8191                17.8, 18.6     17.9, 16.9    19.0, 19.8    17.8, 24.6
// and single tokens of 32 / 8 heads: 32 ragged sequences of up to 8191 115, 102, 32 and 64 equal ones 129, 130
// and 231, 240.  A longer sequence in the call sends its single tokens to few_rows too: 32 ragged ones (of
// 268 MB, which the caches hold in part) and a chunk of 40 over 4096 137 us in one call, 69 and 35 in two.
inline bool codes_call(int dtype, int page_dtype, int64_t max_new, int64_t g, int d) {
  const bool held = page_dtype == SSA_DTYPE_I8 || page_dtype == SSA_DTYPE_E4M3;
  return held && dtype == SSA_DTYPE_BF16 && max_new <= 2 && max_new * g <= 16 && (d <= 64 || d % 16 == 0);
}

// Parts, tiles and workspace of a call.
struct PagedPlan {
  int few_splits, row_splits, row_tiles, row_kw;
  int64_t few_len, row_len;
  size_t few_o, few_ml, row_o, row_ml, bytes;
};

// whole_tiles: parts of the keys of many rows are multiples of as many; codes: few_codes takes the call.
inline PagedPlan paged_plan(int dtype, int64_t tokens, int64_t batch, int h_q, int h_kv, int d, int64_t max_new, int64_t max_len,
                            int64_t whole_tiles = 64, bool codes = false) {
  PagedPlan l{};
  max_new = max_new < tokens ? max_new : tokens;
  const int64_t g = h_q / h_kv, D = d <= 64 ? 64 : 128;
  // Few rows: parts of at least 256 keys, enough for two blocks a CU twice over
  // where the batch has sequences of unlike lengths to even out, once for one.
  const int64_t blocks = batch * h_kv;
  // (few_codes runs three blocks a CU: 1536 of them take 0.88 of 1024's time for 32 ragged sequences of int8,
  // 0.93 for 32 of 8191 tokens, 2048 or more the same or worse)
  int64_t s = div_up(batch > 1 ? (codes ? 1536 : 1024) : 512, blocks), most = div_up(max_len, 256);
  s = s < most ? s : most;
  s = s > 1 ? s : 1;
  l.few_len = div_up(div_up(max_len, s), 128) * 128;
  l.few_splits = static_cast<int>(div_up(max_len, l.few_len));
  l.row_splits = 1;
  l.row_len = 0;
  if (max_new * g > kFew) {
    const int64_t each = batch * max_new, rows = (tokens < each ? tokens : each) * g;
    const DenseSplit cut = dense_split(rows, h_kv, max_len, max_new, dtype == SSA_DTYPE_F32, d > 64, true);
    const int block = 128 / cut.kw;
    // (a sequence's last block may be part empty)
    const int64_t by_seq = batch * div_up(max_new * g, block), ragged = rows / block + batch;
    l.row_kw = cut.kw;
    l.row_tiles = static_cast<int>(by_seq < ragged ? by_seq : ragged);
    l.row_splits = cut.parts;
    l.row_len = div_up(div_up(max_len, l.row_splits), whole_tiles) * whole_tiles;
  }
  if (l.few_splits > 1) {
    const size_t rows = static_cast<size_t>(l.few_splits) * batch * h_kv * kFew;
    l.few_o = l.bytes;
    l.few_ml = l.few_o + rows * D * sizeof(float);
    l.bytes = (l.few_ml + rows * 2 * sizeof(float) + 15) / 16 * 16;
  }
  if (l.row_splits > 1) {
    const size_t rows = static_cast<size_t>(l.row_splits) * tokens * h_q;
    l.row_o = l.bytes;
    l.row_ml = l.row_o + rows * D * sizeof(float);
    l.bytes = (l.row_ml + rows * 2 * sizeof(float) + 15) / 16 * 16;
  }
  return l;
}

}  // namespace ssa
