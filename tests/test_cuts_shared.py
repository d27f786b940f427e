"""The rules of ssa_cuts.h that kernels follow too, through the very functions that they call: the list of
blocks that the backward of two intervals makes of its counts, and the tiles that windowed rows walk."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = r"""
#include <stdio.h>
#include <stdlib.h>
#include <algorithm>
#include <numeric>
#include <vector>
#include "ssa_cuts.h"
using namespace ssa;
#define CHECK(x) do { if (!(x)) { printf("%s, case %d\n", #x, it); return 1; } } while (0)
int main() {
  srand(11);
  int planned = 0, bigs = 0, lefts = 0, ones = 0, unsorted = 0, empty = 0;
  for (int it = 0; it < 30000; ++it) {
    const int64_t n = 1 + rand() % (1 << (1 + rand() % 16)), batch = 1 + rand() % (rand() % 20 ? 4 : 2500);
    const int h_kv = 1 + rand() % (rand() % 3 ? 9 : 40), g = 1 + rand() % 8, d = 8 * (1 + rand() % 16), dtype = rand() % 2;
    const BwdCut b = bwd_cut(dtype, batch, n, n, h_kv * g, h_kv, d);
    const TwoCut t = two_cut(b, dtype, batch, n, h_kv, d);
    if (!t.planned || t.key_blocks > 20000) continue;
    ++planned;
    const int N = static_cast<int>(t.key_blocks), slots = t.slots, most = t.most;
    const int qt = 32 << rand() % 3, sg = qt / 32, tiles = (b.groups + sg - 1) / sg, least = qt < 128 ? 128 / qt : 1;
    const int kind = rand() % 6;
    std::vector<int> h(N);
    for (int x = 0; x < N; ++x) {
      const int some = rand() % (tiles / 9 + 1);
      h[x] = kind == 0 ? tiles : kind == 1 ? rand() % (tiles + 1) : kind == 2 ? (rand() % 50 ? some : tiles) : kind == 3 ? (rand() % 3 ? 0 : some)
             : kind == 4 ? std::min(tiles, 1 + rand() % 3) : (x % 40 ? std::min(tiles, 5 + rand() % 4) : tiles);
    }
    const int64_t total = std::accumulate(h.begin(), h.end(), int64_t(0)), share = plan_share(total, slots, least);
    int64_t big = 0;
    int n_big = 0;
    for (int x : h)
      if (x > share) { big += x; ++n_big; }
    const int P = plan_part(big, t.extra, least, share), one = N - n_big, left = plan_left(N, one, slots), whole = one - left;
    CHECK(P >= 1 && left >= 0 && whole >= 0);
    std::vector<int> order;
    for (int x = 0; x < N; ++x)
      if (h[x] <= share) order.push_back(x);
    if (N <= kSorted) std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return h[x] > h[y]; });
    int64_t sum = 0;
    for (int i = whole; i < one; ++i) sum += h[order[i]];
    const int P2 = left ? plan_left_part(sum, slots, least) : P;
    // the list: what each of its places holds, and the slots of the workspace that parts write to
    std::vector<int> place(N + most, -1), seen(N, 0);
    for (int i = 0; i < whole; ++i) { place[i] = order[i]; ++seen[order[i]]; }
    std::vector<char> late(N, 0);
    for (int i = whole; i < one; ++i) late[order[i]] = 1;
    int from = 0, cut = 0;
    for (int x = 0; x < N; ++x) {
      const bool is_big = h[x] > share;
      if (!is_big && !late[x]) continue;
      const int parts = plan_parts(h[x], is_big ? P : P2);
      CHECK(parts >= 1 && (h[x] == 0 || parts <= h[x]) && int64_t(parts) * (is_big ? P : P2) >= h[x]);
      ones += parts == 1;
      empty += h[x] == 0;
      for (int y = 0; y < parts; ++y) {
        CHECK(whole + from + y < N + most && place[whole + from + y] == -1);
        place[whole + from + y] = x;
      }
      ++seen[x];
      from += parts;
      ++cut;
    }
    for (int x = 0; x < N; ++x) CHECK(seen[x] == 1);
    const int64_t block = int64_t(h_kv) * 32 * b.key_groups * (d > 64 ? 128 : 64);
    CHECK(from <= most && from * block <= int64_t(t.part_floats) && cut <= 2 * slots);
    CHECK(t.counts + 4 * size_t(N) <= t.entries && t.entries + 16 * size_t(N + most) <= t.cut);
    CHECK(t.cut + 16 * size_t(2 * slots + 1) <= t.part && t.part + 8 * t.part_floats <= t.bytes && t.entries % 16 == 0 && t.cut % 16 == 0);
    bigs += n_big > 0;
    lefts += left > 0;
    unsorted += N > kSorted;
  }
  if (planned < 3000 || bigs < 300 || lefts < 300 || ones < 300 || unsorted < 30 || empty < 300) {
    printf("planned %d, big %d, last rounds %d, of one part %d, unsorted %d, empty %d\n", planned, bigs, lefts, ones, unsorted, empty);
    return 1;
  }
  printf("ok\n");
  return 0;
}
"""

TILES = r"""
#include <stdio.h>
#include <stdlib.h>
#include <algorithm>
#include <vector>
#include "ssa_cuts.h"
using namespace ssa;
#define CHECK(x) do { if (!(x)) { printf("%s, case %d\n", #x, it); return 1; } } while (0)
// whether the walk is ascending and holds just the tiles that some marked key lies in
static bool right(const Tiles& w, const std::vector<char>& key, int kt, bool none_more) {
  int last = -1;
  std::vector<char> tile((key.size() + kt - 1) / kt + 2, 0);
  for (int t = 0; t < w.n; ++t) {
    const int x = w.at(t);
    if (x <= last || x >= static_cast<int>(tile.size())) return false;
    last = x;
    tile[x] = 1;
  }
  std::vector<char> want(tile.size(), 0);
  for (size_t j = 0; j < key.size(); ++j)
    if (key[j]) want[j / kt] = 1;
  for (size_t x = 0; x < tile.size(); ++x)
    if ((want[x] && !tile[x]) || (none_more && tile[x] && !want[x])) return false;
  return true;
}
int main() {
  srand(12);
  for (int it = 0; it < 60000; ++it) {
    const int len = 1 + rand() % (1 << (1 + rand() % 12)), m = 1 + rand() % (len < 500 ? len : 500), cached = len - m;
    const int window = rand() % 6 ? 1 + rand() % (1 << (1 + rand() % 12)) : 0, sinks = window ? rand() % (1 << (rand() % 11)) : 0;
    const int64_t most = len + rand() % 3 * (rand() % 900), g = 1 + rand() % 8;
    const int page_dtype = rand() % 4, dtype = rand() % 2, d = 8 * (1 + rand() % 16);
    if (window >= most) continue;  // (such a window is none)
    auto mark = [&](int t, int u) {  // the keys that the new tokens t to u see, from the definition
      std::vector<char> key(len, 0);
      for (int p = cached + t; p <= cached + u; ++p)
        for (int j = 0; j <= p; ++j)
          if (!window || p - j < window || j < sinks) key[j] = 1;
      return key;
    };
    const Tiles w = seen_tiles(cached, len, window, sinks, 32);
    if (it % 4 == 0) CHECK(right(w, mark(0, m - 1), 32, true));
    const int64_t batch = 1 + rand() % 5;
    const PagedPlan l = paged_plan(dtype, m * batch, batch, g * 2, 2, d, m, seen_len(most, m, window, sinks), 128,
                                   codes_call(dtype, page_dtype, m, g, d));
    CHECK(w.n * int64_t(32) <= l.few_splits * l.few_len && l.few_len % 128 == 0);
    if (l.row_tiles && l.row_splits > 1) {
      const int t = rand() % m, u = t + rand() % (m - t);
      CHECK(l.row_len % 128 == 0);
      for (int kt = 32; kt <= 128; kt *= 2) {
        // what a block's rows see between them, as dense_rows joins it
        int lo_min = 0x7FFFFFFF, hi_max = 0, a_max = 0;
        for (int p = cached + t; p <= cached + u; ++p) {
          const int lo = window ? std::max(p + 1 - window, 0) : 0;
          lo_min = std::min(lo_min, lo);
          hi_max = std::max(hi_max, p + 1);
          a_max = std::max(a_max, std::min(sinks, lo));
        }
        const Tiles x = tiles_of(0, a_max, lo_min, hi_max, kt);
        if (it % 16 == 0) CHECK(right(x, mark(t, u), kt, true));
        CHECK(x.n * int64_t(kt) <= l.row_splits * l.row_len);
      }
    }
  }
  // any two ranges, in any order
  for (int it = 0; it < 200000; ++it) {
    const int a = rand() % 700, b = a + rand() % 300 - 40, c = rand() % 700, e = c + rand() % 300 - 40, kt = 32 << rand() % 3;
    std::vector<char> key(1100, 0);
    for (int j = 0; j < 1100; ++j) key[j] = (j >= a && j < b) || (j >= c && j < e);
    const Tiles w = b > a ? tiles_of(a, b, e > c ? c : 0, e > c ? e : 0, kt) : tiles_of(0, 0, e > c ? c : 0, e > c ? e : 0, kt);
    CHECK(right(w, key, kt, true));
  }
  printf("ok\n");
  return 0;
}
"""


def build_and_run(source, path):
    src, exe = path / "cuts.cpp", path / "cuts"
    src.write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT}/include", f"-I{ROOT}/ssa_amd/csrc", "-o", str(exe), str(src)],
                   check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True).stdout


def test_the_list_of_the_backward_holds_every_block_once(tmp_path):
    """Of any counts: each block of keys whole or in all its parts, parts in slots of their own, within the
    workspace; with big blocks, a last round that is cut, cut blocks of one part, blocks that nobody sees."""
    assert build_and_run(PLAN, tmp_path) == "ok\n"


def test_windowed_rows_walk_the_tiles_that_they_see(tmp_path):
    """Those and no others, in order, and the parts of a call hold them all."""
    assert build_and_run(TILES, tmp_path) == "ok\n"


CODES = r"""
#include <stdio.h>
#include "ssa_cuts.h"
using namespace ssa;
int main() {
  for (int dtype = 0; dtype < 2; ++dtype)
    for (int page = 0; page < 4; ++page)
      for (int64_t m = 1; m <= 64; ++m)
        for (int64_t g = 1; g <= 32; ++g)
          for (int d = 8; d <= 128; d += 8) {
            const bool want = dtype == SSA_DTYPE_BF16 && page >= 2 && m <= 2 && m * g <= 16 && (d <= 64 || d % 16 == 0);
            if (codes_call(dtype, page, m, g, d) != want) { printf("%d %d %d %d %d\n", dtype, page, int(m), int(g), d); return 1; }
          }
  printf("ok\n");
  return 0;
}
"""


def test_few_codes_takes_one_or_two_tokens(tmp_path):
    """(Sixteen drafts of one head took 13 us by few_rows and 32 by few_codes.)"""
    assert build_and_run(CODES, tmp_path) == "ok\n"
