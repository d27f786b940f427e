"""The planned dK and dV of rows that see two key intervals, branch by branch: which one a case takes is asked of
ssa_cuts.h's rules, with the counts that its mask gives."""

import os
import subprocess

import pytest
import torch

from tests.test_gpu_windows import run, window_sees

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROBE = r"""
#include <stdio.h>
#include <stdlib.h>
#include <algorithm>
#include <vector>
#include "ssa_cuts.h"
using namespace ssa;
// dtype batch n h_q h_kv d: planned, keys of a block; with counts on stdin and the rows of a tile too: blocks that are big,
// that the last round cuts, of those in one part and seen by nobody, parts in all, whether the list is sorted
int main(int, char** a) {
  const int dtype = atoi(a[1]), h_q = atoi(a[4]), h_kv = atoi(a[5]), d = atoi(a[6]);
  const int64_t batch = atoll(a[2]), n = atoll(a[3]);
  const BwdCut b = bwd_cut(dtype, batch, n, n, h_q, h_kv, d);
  const TwoCut t = two_cut(b, dtype, batch, n, h_kv, d);
  const int qt = atoi(a[7]);
  if (qt == 0) { printf("%d %d %d\n", int(t.planned), b.key_groups, t.slots); return 0; }
  const int least = qt < 128 ? 128 / qt : 1;
  std::vector<int> h;
  for (int x; scanf("%d", &x) == 1;) h.push_back(x);
  if (int64_t(h.size()) != t.key_blocks) return 1;
  int64_t total = 0, big = 0, sum = 0;
  int n_big = 0, one_part = 0, nobody = 0, parts = 0;
  for (int x : h) total += x;
  const int64_t share = plan_share(total, t.slots, least);
  std::vector<int> rest;
  for (int x : h) {
    if (x > share) { big += x; ++n_big; } else rest.push_back(x);
  }
  std::sort(rest.rbegin(), rest.rend());
  const int P = plan_part(big, t.extra, least, share), left = plan_left(h.size(), rest.size(), t.slots);
  for (size_t i = rest.size() - left; i < rest.size(); ++i) sum += rest[i];
  for (size_t i = rest.size() - left; i < rest.size(); ++i) {
    const int y = plan_parts(rest[i], plan_left_part(sum, t.slots, least));
    parts += y;
    one_part += y == 1 && rest[i] > 0;
    nobody += rest[i] == 0;
  }
  for (int x : h)
    if (x > share) parts += plan_parts(x, P);
  printf("%d %d %d %d %d %d\n", n_big, left, one_part, nobody, parts, int(h.size()) <= kSorted);
  return 0;
}
"""


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    path = tmp_path_factory.mktemp("plan")
    (path / "plan.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT}/include", f"-I{ROOT}/ssa_amd/csrc", "-o", str(path / "plan"),
                    str(path / "plan.cpp")], check=True)

    def ask(dtype, batch, n, h_q, h_kv, d, qt=0, counts=()):
        res = subprocess.run([str(path / "plan"), *map(str, (int(dtype == BF16), batch, n, h_q, h_kv, d, qt))],
                             input=" ".join(map(str, counts)), capture_output=True, text=True, check=True)
        return [int(x) for x in res.stdout.split()]

    return ask


def plan_of(probe, dtype, spans, n, h_q, h_kv, d):
    """What the plan makes of the spans [B, n, 4] (on the host)."""
    B, g = len(spans), h_q // h_kv
    planned, groups, slots = probe(dtype, B, n, h_q, h_kv, d)
    if not planned:
        return None
    # rows of a tile (DkvShape): waves that take rows in turn, of 32 rows each, of bf16 alone 64
    waves = {4: 2 if dtype == BF16 and d > 64 else 1, 2: 2, 1: 4}[groups]
    qt = 32 * waves * (2 if waves == 1 and dtype == BF16 else 1)
    counts = []
    for x in spans.long():
        rows = x.repeat_interleave(g, 0)
        pad = -len(rows) % qt
        rows = torch.cat([rows, torch.zeros(pad, 4, dtype=torch.long)]).clamp(0, n)
        one, two = rows[:, 1] > rows[:, 0], rows[:, 3] > rows[:, 2]
        a, z, x, y = rows.unbind(1)
        # (one interval alone is the first)
        a, z = torch.where(one, a, x), torch.where(one, z, y)
        some, both = one | two, one & two
        hull = lambda lo, hi, on: (torch.where(on, lo, 1 << 30).view(-1, 32).amin(1), torch.where(on, hi, 0).view(-1, 32).amax(1))  # noqa: E731
        (a, z), (x, y) = hull(a, z, some), hull(x, y, both)
        for k0 in range(0, n, 32 * groups):
            hit = ((a < k0 + 32 * groups) & (z > k0)) | ((x < k0 + 32 * groups) & (y > k0))
            counts.append(int(hit.view(-1, qt // 32).any(1).sum()))
    big, left, one_part, nobody, parts, is_sorted = probe(dtype, B, n, h_q, h_kv, d, qt, counts)
    return dict(blocks=len(counts), slots=slots, big=big, left=left, one_part=one_part, nobody=nobody, parts=parts, sorted=is_sorted,
                empty=counts.count(0))


def draw(seed, dtype, B, n, h_q, h_kv, d):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, n, h, d, generator=g).to(dtype) for h in (h_q, h_kv, h_kv, h_q)]


CASES = {
    # dtype, B, n, h_q, h_kv, d, window, sinks, starts, cap, bias, what the plan has to hold
    "bf16 d=128, groups of 4, padded documents": (BF16, 2, 700, 32, 8, 128, 90, 5, [[0, 250, 600], [30, 31, 690]], 0.0, False,
                                                  lambda x: x["big"] > 0),
    "bf16 d=128, first keys seen by all": (BF16, 1, 1500, 8, 8, 128, 40, 7, None, 0.0, True, lambda x: x["big"] > 0 and x["parts"] > x["big"]),
    "bf16 d=128, a last round that is cut": (BF16, 7, 380, 32, 16, 128, 100, 0, [[0, 380], [0, 379], [1, 380], [0, 375], [0, 378], [5, 380], [0, 370]],
                                             0.0, False, lambda x: x["left"] > 0 and x["parts"] > x["left"] + 2 and x["big"] == 0),
    "bf16 d=128, a last round that nobody sees": (BF16, 6, 400, 16, 16, 128, 100, 1, [[0, 400], [0, 100], [10, 350], [0, 385], [0, 50], [5, 200]],
                                                  0.0, True, lambda x: x["left"] > 0 and x["nobody"] > 0),
    "bf16 d=128, a last round of one part a block": (BF16, 6, 500, 16, 16, 128, 30, 0, None, 3.0, False,
                                                     lambda x: x["left"] > 0 and x["one_part"] > 0),
    "bf16 d=128, far caps and bias": (BF16, 3, 640, 16, 8, 128, 130, 64, [[0, 300, 640], [10, 20, 600], [0, 640, 640]], 900.0, True,
                                      lambda x: x["big"] > 0),
    "bf16 d=72, groups of 7": (BF16, 2, 1100, 28, 4, 72, 50, 130, [[0, 515], [60, 1090]], 0.0, False, lambda x: x["blocks"] > 0),
    "bf16 d=64": (BF16, 2, 1030, 16, 8, 64, 64, 3, [[0, 500, 1030], [7, 900, 900]], 0.0, True, lambda x: x["big"] > 0),
    "bf16 d=64, a last round that is cut": (BF16, 3, 900, 32, 32, 64, 33, 2, [[0, 450, 900], [0, 40, 200], [880, 890, 900]], 0.0, False,
                                            lambda x: x["left"] > 0 and x["nobody"] > 0),
    "fp32 d=64": (F32, 2, 1100, 16, 8, 64, 77, 9, [[0, 333, 1099], [0, 1100, 1100]], 0.0, False, lambda x: x["big"] > 0),
    "fp32 d=128, a last round that is cut": (F32, 3, 900, 32, 32, 128, 60, 4, [[0, 450, 900], [0, 40, 200], [3, 890, 900]], 2.0, True,
                                             lambda x: x["left"] > 0),
}


@pytest.mark.parametrize("name", CASES)
def test_planned_gradients(dev, probe, name):
    """Every value and gradient against the oracle; rows and keys of no document hold NaN and infinities, so that
    the blocks that they share are computed again pair by pair, cut ones into their slots."""
    from ssa_amd import mask_spans

    dtype, B, n, h_q, h_kv, d, window, sinks, starts, cap, bias, holds = CASES[name]
    spans = mask_spans(n, B, doc_starts=None if starts is None else torch.tensor(starts, device=dev), window=window, sinks=sinks, device=dev)
    plan = plan_of(probe, dtype, spans.cpu(), n, h_q, h_kv, d)
    print(name, plan, flush=True)
    assert plan is not None and holds(plan), plan
    q, k, v, dout = draw(91, dtype, B, n, h_q, h_kv, d)
    see = torch.stack([window_sees(n, n, 0, window, sinks, starts and starts[b]) for b in range(B)])
    slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)]) if bias else None
    run(dev, q, k, v, spans, see, 0, cap, slopes, dout)
    if starts is None:
        return
    alone, unseen = ~see.any(2), ~see.any(1)  # rows without a key, keys without a row
    assert alone.any() and unseen.any()
    for t, where, x in ((q, alone, float("nan")), (dout, alone, float("inf")), (k, unseen, float("inf")), (v, unseen, float("nan"))):
        t[where] = x
    got = run(dev, q, k, v, spans, see, 0, cap, slopes, dout)
    assert not got["dq"][alone].any() and not got["dk"][unseen].any() and not got["dv"][unseen].any()


def test_a_list_too_long_to_sort(dev, probe):
    """More than 2048 blocks of keys, of unlike documents: an element of the batch is what it is by itself."""
    from ssa_amd import mask_spans

    B, n, h, d, window, sinks = 1100, 150, 1, 64, 12, 2
    starts = [[0, i % 149, 150 - i % 7] for i in range(B)]
    spans = mask_spans(n, B, doc_starts=torch.tensor(starts, device=dev), window=window, sinks=sinks, device=dev)
    plan = plan_of(probe, BF16, spans.cpu(), n, h, h, d)
    print(plan, flush=True)
    assert plan is not None and not plan["sorted"] and plan["left"] == 0
    q, k, v, dout = draw(92, BF16, B, n, h, h, d)
    see = torch.stack([window_sees(n, n, 0, window, sinks, x) for x in starts])
    run(dev, q, k, v, spans, see, 0, dout=dout)


def test_planned_calls_captured_and_on_streams(dev, probe):
    """Same bits on every stream and on every replay, beside eager calls of other inputs."""
    from ssa_amd import mask_spans, masked_attention

    B, n, h_q, h_kv, d = 2, 700, 16, 8, 128
    starts = torch.tensor([[0, 250, 600], [30, 31, 690]], device=dev)
    q, k, v, dout = draw(93, BF16, B, n, h_q, h_kv, d)
    x = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    dout = dout.to(dev)

    def step():
        spans = mask_spans(n, B, doc_starts=starts, window=90, sinks=5, device=dev)
        out = masked_attention(*x, spans)
        return (out.detach(), *torch.autograd.grad(out, x, dout))

    plan = plan_of(probe, BF16, mask_spans(n, B, doc_starts=starts, window=90, sinks=5, device=dev).cpu(), n, h_q, h_kv, d)
    assert plan is not None and plan["big"] > 0
    want = step()
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for st in streams * 3:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for y in got for a, b in zip(y, want))
    del got
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(4):
        with torch.no_grad():
            x[0].add_(0.1)
        if i == 2:  # (the documents are read by the kernels: a replay follows them)
            starts.copy_(torch.tensor([[0, 400, 700], [0, 10, 300]], device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, step()))
