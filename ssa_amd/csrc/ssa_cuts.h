// How the dense attention calls are cut into blocks, and the workspaces that follow: host
// rules on sizes and types alone, in plain C++, so that a host test can ask for a call's cut.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "ssa_hip.h"

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

// Parts, tiles and workspace of a call.
struct PagedPlan {
  int few_splits, row_splits, row_tiles, row_kw;
  int64_t few_len, row_len;
  size_t few_o, few_ml, row_o, row_ml, bytes;
};

inline PagedPlan paged_plan(int dtype, int64_t tokens, int64_t batch, int h_q, int h_kv, int d, int64_t max_new, int64_t max_len) {
  PagedPlan l{};
  max_new = max_new < tokens ? max_new : tokens;
  const int64_t g = h_q / h_kv, D = d <= 64 ? 64 : 128;
  // Few rows: parts of at least 256 keys, enough for two blocks a CU twice over
  // where the batch has sequences of unlike lengths to even out, once for one.
  const int64_t blocks = batch * h_kv;
  int64_t s = div_up(batch > 1 ? 1024 : 512, blocks), most = div_up(max_len, 256);
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
    l.row_len = div_up(div_up(max_len, l.row_splits), 64) * 64;
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
