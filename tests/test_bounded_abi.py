"""Host-side checks of the windowed, tree and 8-bit cache entry points: every call here fails
validation or is an empty no-op, so nothing is launched and no pointer is dereferenced."""

import ctypes
import os
import subprocess

import pytest
import torch

import ssa_amd
from ssa_amd import _lib

FAKE = ctypes.c_void_p(1 << 20)
ODD8 = ctypes.c_void_p((1 << 20) + 8)
ODD4 = ctypes.c_void_p((1 << 20) + 4)
ODD1 = ctypes.c_void_p((1 << 20) + 1)
OK, INVALID, UNSUPPORTED, WORKSPACE = (_lib.SSA_OK, _lib.SSA_ERR_INVALID_ARGUMENT, _lib.SSA_ERR_UNSUPPORTED,
                                       _lib.SSA_ERR_WORKSPACE)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libssa_hip.so not built (run __graft_entry__.build())")
    return _lib.load()


def call(L, name, defaults, kw):
    a = {**defaults, **kw}
    assert set(a) == set(defaults)
    st = getattr(L, name)(*a.values())
    return st, (L.ssa_last_error() or b"").decode()


STEP = dict(q=FAKE, k=FAKE, v=FAKE, dtype=_lib.DTYPE_BF16, tokens=10, batch=3, h_q=8, h_kv=2, d=64, q_st=512, q_sh=64,
            k_st=128, k_sh=64, v_st=128, v_sh=64, k_pages=FAKE, v_pages=FAKE, page_dtype=_lib.DTYPE_I8, k_scales=FAKE,
            v_scales=FAKE, num_pages=100, page_size=16, kp_sp=2048, kp_st=128, kp_sh=64, vp_sp=2048, vp_st=128, vp_sh=64,
            ks_sp=32, ks_st=2, ks_sh=1, vs_sp=32, vs_st=2, vs_sh=1, table=FAKE, table_stride=64, max_pages=64, starts=FAKE,
            cached=FAKE, parents=None, max_new=8, max_len=1000, window=0, sinks=0, scale=8.0, cap=0.0, slopes=None, out=FAKE,
            o_st=512, o_sh=64, zero_rows=0, flag=None, ws=FAKE, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=_lib.DTYPE_I8), UNSUPPORTED, "dtype"), (dict(page_dtype=7), UNSUPPORTED, "pages hold"),
    (dict(page_dtype=_lib.DTYPE_F32), UNSUPPORTED, "pages hold"), (dict(h_q=9), INVALID, "divisible"),
    (dict(h_q=34), UNSUPPORTED, "group"), (dict(d=60), UNSUPPORTED, "head_dim"), (dict(tokens=-1), INVALID, "shape"),
    (dict(page_size=24), UNSUPPORTED, "page_size"), (dict(window=-1), INVALID, "window"), (dict(sinks=-1, window=4), INVALID, "sinks"),
    (dict(sinks=3), INVALID, "sinks"), (dict(k_scales=None), INVALID, "scales"), (dict(v_scales=ODD1), INVALID, "scales"),
    (dict(ks_st=-2), INVALID, "strides"), (dict(k_pages=ODD4), UNSUPPORTED, "k_pages"), (dict(vp_st=132), UNSUPPORTED, "v_pages"),
    (dict(kp_sp=-2048), UNSUPPORTED, "strides"), (dict(kp_st=1 << 25), UNSUPPORTED, "strides"),
    (dict(page_dtype=_lib.DTYPE_BF16, k_pages=ODD8), UNSUPPORTED, "k_pages"), (dict(table=None), INVALID, "null"),
    (dict(k=None), INVALID, "null"), (dict(parents=FAKE, tokens=100, max_new=65), UNSUPPORTED, "64"),
    (dict(parents=FAKE, tokens=100, max_new=99), UNSUPPORTED, "64"), (dict(scale=0.0), INVALID, "scale"),
    (dict(cap=float("nan")), INVALID, "softcap"), (dict(q=ODD8), UNSUPPORTED, "q must"), (dict(o_st=4), UNSUPPORTED, "out must"),
    (dict(ws=None), WORKSPACE, "workspace"), (dict(ws_bytes=100), WORKSPACE, "workspace"), (dict(ws=ODD8), INVALID, "workspace"),
    (dict(batch=0, q=None, zero_rows=1), INVALID, "without a sequence"), (dict(tokens=0, q=None), OK, ""),
    (dict(batch=0, q=None), OK, ""), (dict(max_new=0), INVALID, "max_new"), (dict(tokens=1 << 30), UNSUPPORTED, "2^31"),
])
def test_step(L, kw, status, text):
    st, msg = call(L, "ssa_paged_step_general", STEP, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("kw", [dict(), dict(max_new=1), dict(max_new=1 << 62), dict(max_len=1 << 30), dict(window=300), dict(window=1 << 62, sinks=1 << 62),
                                dict(window=1, sinks=(1 << 31) - 1), dict(dtype=_lib.DTYPE_F32), dict(page_dtype=_lib.DTYPE_E4M3, d=72, h_q=2),
                                dict(tokens=700, batch=16, max_new=300), dict(page_dtype=_lib.DTYPE_BF16, window=64, tokens=500, batch=1, max_new=500, max_len=9000)])
def test_step_workspace(L, kw):
    a = {**STEP, **kw}
    need = L.ssa_paged_step_general_workspace_bytes(*[a[x] for x in ("dtype", "page_dtype", "tokens", "batch", "h_q", "h_kv", "d",
                                                                     "max_new", "max_len", "window", "sinks")])
    if need:
        for ws, have in ((FAKE, need - 1), (None, need)):
            st, msg = call(L, "ssa_paged_step_general", STEP, dict(kw, ws=ws, ws_bytes=have))
            assert st == WORKSPACE and f"workspace of {need} bytes" in msg, msg


def test_workspaces_of_sizes_that_no_call_takes(L):
    f = L.ssa_paged_step_general_workspace_bytes
    assert f(1, 2, 1 << 62, 3, 8, 2, 64, 8, 1000, 0, 0) == 0 and f(1, 2, 10, 1 << 62, 8, 2, 64, 8, 1000, 0, 0) == 0
    assert f(1, 2, 10, 3, 8, 2, 64, 8, 1 << 62, 1 << 62, 1 << 62) == 0 and f(1, 2, 10, 3, 8, 0, 64, 8, 1000, 0, 0) == 0
    assert f(1, 2, 10, 3, 8, 2, 64, -1, 1000, 0, 0) == 0 and f(1, 2, 10, 3, 8, 2, 64, 8, 1000, -1, 0) == 0
    g = L.ssa_masked_attention_two_backward_workspace_bytes
    assert g(1, 1 << 40, 100, 100, 8, 2, 64) == 0 and g(1, 1, 1 << 40, 100, 8, 2, 64) == 0 and g(1, 1, 100, 100, 8, 3, 64) == 0
    assert g(1, 1, 100, 100, 8, 2, 64) > 0


POOL = dict(k_pages=FAKE, v_pages=FAKE, page_dtype=_lib.DTYPE_I8, k_scales=FAKE, v_scales=FAKE, num_pages=100, page_size=16, h_kv=2,
            d=64, kp_sp=2048, kp_st=128, kp_sh=64, vp_sp=2048, vp_st=128, vp_sh=64, ks_sp=32, ks_st=2, ks_sh=1, vs_sp=32, vs_st=2,
            vs_sh=1, batch=3, table=FAKE, table_stride=64, max_pages=64)
READ = dict(**POOL, starts=FAKE, first=FAKE, tokens=10, out_dtype=_lib.DTYPE_BF16, k_out=FAKE, v_out=FAKE, flag=None, stream=None)
KEEP = dict(**POOL, cached=FAKE, kept=FAKE, kept_stride=8, most=8, flag=None, stream=None)
POOLS = [
    (dict(page_dtype=4), UNSUPPORTED, "pages hold"), (dict(d=60), UNSUPPORTED, "head_dim"), (dict(d=136), UNSUPPORTED, "head_dim"),
    (dict(page_size=12), UNSUPPORTED, "page_size"), (dict(h_kv=0), INVALID, "shape"), (dict(k_pages=None), INVALID, "null"),
    (dict(v_scales=None), INVALID, "null"), (dict(kp_st=4), UNSUPPORTED, "k_pages"), (dict(vp_sh=-64), UNSUPPORTED, "strides"),
    (dict(ks_sh=-1), UNSUPPORTED, "strides"), (dict(table=None), INVALID, "null"), (dict(max_pages=1 << 28), UNSUPPORTED, "2^31"),
    (dict(num_pages=0), INVALID, "num_pages"), (dict(batch=-1), INVALID, "shape"),
]


@pytest.mark.parametrize("kw,status,text", POOLS + [
    (dict(out_dtype=_lib.DTYPE_I8), UNSUPPORTED, "8 bits"), (dict(page_dtype=_lib.DTYPE_F32), UNSUPPORTED, "pages' type"),
    (dict(tokens=-1), INVALID, "tokens"), (dict(first=None), INVALID, "null"), (dict(v_out=ODD8), UNSUPPORTED, "outputs"),
    (dict(tokens=0, k_pages=None), OK, ""), (dict(batch=0), INVALID, "batch"),
])
def test_read(L, kw, status, text):
    st, msg = call(L, "ssa_paged_read", READ, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("kw,status,text", POOLS + [
    (dict(most=65), UNSUPPORTED, "64"), (dict(most=-1), INVALID, "most_kept"), (dict(kept=None), INVALID, "null"),
    (dict(cached=None), INVALID, "null"), (dict(most=0, table=None), OK, ""), (dict(batch=0, table=None), OK, ""),
    (dict(page_dtype=_lib.DTYPE_F32, k_pages=ODD8), UNSUPPORTED, "16 bytes"),
])
def test_keep(L, kw, status, text):
    st, msg = call(L, "ssa_paged_keep", KEEP, kw)
    assert st == status and (st == OK or text in msg), msg


SPANS = dict(starts=FAKE, docs=3, prefix=FAKE, batch=2, n=100, n_q=100, q_pos0=0, window=8, sinks=2, spans=FAKE, stream=None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(window=0), INVALID, "window"), (dict(sinks=-1), INVALID, "sinks"), (dict(n=-1), INVALID, "shape"),
    (dict(docs=0), INVALID, "docs"), (dict(starts=None), INVALID, "one document"), (dict(spans=None), INVALID, "null"),
    (dict(spans=ODD8), INVALID, "16 bytes"), (dict(batch=0, spans=None), OK, ""),
])
def test_mask_spans_window(L, kw, status, text):
    st, msg = call(L, "ssa_mask_spans_window", SPANS, kw)
    assert st == status and (st == OK or text in msg), msg


def test_two_intervals_want_aligned_spans(L):
    rows = {f"{x}_{s}": v for x in "qkv" for s, v in (("sb", 64000 * 8), ("sn", 512), ("sh", 64))}
    heads = dict(dtype=_lib.DTYPE_BF16, batch=1, n=1000, n_q=1000, q_pos0=0, h_q=8, h_kv=2, d=64)
    fwd = dict(q=FAKE, k=FAKE, v=FAKE, **heads, **rows, spans=FAKE, scale=8.0, cap=0.0, slopes=None, out=FAKE, o_sb=0, o_sn=512,
               o_sh=64, out_low=None, lse=None, ws=FAKE, ws_bytes=1 << 30, stream=None)
    bwd = dict(q=FAKE, k=FAKE, v=FAKE, **heads, **rows, spans=FAKE, scale=8.0, cap=0.0, slopes=None, out=FAKE, out_low=None, o_sb=0,
               o_sn=512, o_sh=64, dout=FAKE, do_sb=0, do_sn=512, do_sh=64, lse=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, ws=FAKE,
               ws_bytes=1 << 40, stream=None)
    for name, args in (("ssa_masked_attention_two", fwd), ("ssa_masked_attention_two_backward", bwd)):
        for spans in (None, ODD8):
            st, msg = call(L, name, args, dict(spans=spans))
            assert st == INVALID and "spans" in msg
        st, msg = call(L, name, args, dict(d=60))
        assert st == UNSUPPORTED and name in msg
    need = L.ssa_masked_attention_two_backward_workspace_bytes(_lib.DTYPE_BF16, 1, 1000, 1000, 8, 2, 64)
    st, msg = call(L, "ssa_masked_attention_two_backward", bwd, dict(ws_bytes=need - 1))
    assert st == WORKSPACE and str(need) in msg


CUTS = r"""
#include <stdio.h>
#include <stdlib.h>
#include "ssa_cuts.h"
using namespace ssa;
// the tiles of kt keys that rows at positions [first, last] see, as the kernels walk them
static int64_t tiles(int64_t first, int64_t last, int64_t window, int64_t sinks, int64_t kt) {
  const int64_t lo = first + 1 - window > 0 ? first + 1 - window : 0, far = last + 1 - window > 0 ? last + 1 - window : 0;
  const int64_t a = sinks < far ? sinks : far;
  int64_t x1 = (a + kt - 1) / kt, y0 = lo / kt, y1 = (last + kt) / kt;
  return y0 <= x1 ? y1 : x1 + y1 - y0;
}
int main() {
  srand(5);
  for (int it = 0; it < 200000; ++it) {
    const int64_t len = 1 + rand() % (1 << (1 + rand() % 16)), m = 1 + rand() % (len < 700 ? len : 700);
    const int64_t window = 1 + rand() % (1 << (1 + rand() % 15)), sinks = rand() % (1 << (rand() % 12));
    const int64_t most = len + rand() % 3 * (rand() % 900), g = 1 + rand() % 8;
    const int page_dtype = rand() % 4, dtype = rand() % 2, d = 8 * (1 + rand() % 16);
    if (window >= most) continue;  // (such a window is none)
    const int64_t batch = 1 + rand() % 5;
    const PagedPlan l = paged_plan(dtype, m * batch, batch, g * 2, 2, d, m, seen_len(most, m, window, sinks), 128,
                                   codes_call(dtype, page_dtype, m, g, d));
    if (tiles(len - m, len - 1, window, sinks, 32) * 32 > l.few_splits * l.few_len || l.few_len % 128) { printf("few %d\n", it); return 1; }
    if (l.row_tiles && l.row_splits > 1) {
      if (l.row_len % 128) { printf("length %d\n", it); return 1; }
      const int64_t t = rand() % m, u = t + rand() % (m - t);
      for (int64_t kt = 32; kt <= 128; kt *= 2)
        if (tiles(len - m + t, len - m + u, window, sinks, kt) * kt > l.row_splits * l.row_len) { printf("rows %d\n", it); return 1; }
    }
  }
  // parts and slots of the backward of two intervals: what plan_list_kernel may make of any counts
  for (int it = 0; it < 20000; ++it) {
    const int64_t n = 1 + rand() % (1 << (1 + rand() % 16)), batch = 1 + rand() % 3;
    const int h_kv = 1 + rand() % 9, g = 1 + rand() % 8, d = 8 * (1 + rand() % 16), dtype = rand() % 2;
    const BwdCut b = bwd_cut(dtype, batch, n, n, h_kv * g, h_kv, d);
    const TwoCut t = two_cut(b, dtype, batch, n, h_kv, d);
    const int64_t qt = 32 << rand() % 3, sg = qt / 32, most_tiles = (b.groups + sg - 1) / sg, least = qt < 128 ? 128 / qt : 1;
    int64_t total = 0, big = 0, n_big = 0;
    static int64_t h[100000];
    if (t.key_blocks > 100000) continue;
    const int kind = rand() % 4;
    for (int64_t x = 0; x < t.key_blocks; ++x) {
      h[x] = kind == 0 ? most_tiles : kind == 1 ? rand() % (most_tiles + 1) : rand() % 50 ? rand() % (most_tiles / 9 + 1) : most_tiles;
      total += h[x];
    }
    int64_t share = (total + t.slots - 1) / t.slots;
    if (share < least) share = least;
    for (int64_t x = 0; x < t.key_blocks; ++x)
      if (h[x] > share) { big += h[x]; ++n_big; }
    int64_t P = (big + t.extra - 1) / t.extra;
    if (P < least) P = least;
    if (P < share / 10) P = share / 10;
    int64_t parts = 0, cut = 0;
    const int64_t n_one = t.key_blocks - n_big, left = n_one % t.slots;
    const bool cut_left = t.key_blocks <= 2048 && n_one > t.slots && n_one < 4 * t.slots && left > 0 && 10 * left < 7 * t.slots;
    for (int64_t x = 0; x < t.key_blocks; ++x)
      if (h[x] > share) { parts += (h[x] + P - 1) / P; ++cut; }
    if (cut_left) {  // (at most one part a slot beyond one a block)
      parts += t.slots + left;
      cut += left;
    }
    // a part less for every block that is cut stands in the list's place for that block
    if (parts - cut > t.most || cut > 2 * t.slots) { printf("list %d\n", it); return 1; }
    const int64_t all = t.key_blocks * b.groups, room = all < t.most ? all : t.most;
    if (!cut_left && parts > room) { printf("slots %d: %lld of %lld\n", it, (long long)parts, (long long)room); return 1; }
    if (cut_left && t.most <= all && parts > t.most) { printf("slots %d: %lld of %d\n", it, (long long)parts, t.most); return 1; }
  }
  printf("ok\n");
  return 0;
}
"""


def test_cuts_hold_what_the_kernels_walk(tmp_path):
    """Parts of a windowed step hold every tile that its rows see; the backward's plan stays within its lists."""
    src, exe = tmp_path / "cuts.cpp", tmp_path / "cuts"
    src.write_text(CUTS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT}/include", f"-I{ROOT}/ssa_amd/csrc", "-o", str(exe), str(src)],
                   check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "ok\n"


def test_python_refuses():
    z = torch.zeros
    q, k = z(3, 4, 64, dtype=torch.bfloat16), z(3, 2, 64, dtype=torch.bfloat16)
    pages = z(5, 16, 2, 64, dtype=torch.bfloat16)
    table, starts, cached = z(1, 5, dtype=torch.int32), z(2, dtype=torch.int32), z(1, dtype=torch.int32)
    args = (q, k, k, pages, pages.clone(), table, starts, cached)
    with pytest.raises(ValueError, match="window"):
        ssa_amd.paged_step(*args, window=0)
    with pytest.raises(ValueError, match="sinks"):
        ssa_amd.paged_step(*args, sinks=3)
    with pytest.raises(ValueError, match="sinks"):
        ssa_amd.paged_step(*args, window=5, sinks=-1)
    with pytest.raises(RuntimeError, match="GPU"):
        ssa_amd.paged_step(*args, window=5)
    with pytest.raises(RuntimeError, match="GPU"):
        ssa_amd.paged_read(pages, pages, table, starts, cached, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        ssa_amd.paged_keep(pages, pages, table, cached, z(1, 2, dtype=torch.int32))
    leaf = pages.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="gradient"):
        ssa_amd.paged_read(leaf, leaf, table, starts, cached, 3)
    with pytest.raises(NotImplementedError, match="gradient"):
        ssa_amd.paged_keep(leaf, leaf, table, cached, z(1, 2, dtype=torch.int32))
    with pytest.raises(NotImplementedError, match="gradient"):
        ssa_amd.paged_step(*args, k_scales=z(5, 16, 2).requires_grad_(True))
    with pytest.raises(ValueError, match="window"):
        ssa_amd.mask_spans(10, window=0)
    with pytest.raises(ValueError, match="causal"):
        ssa_amd.mask_spans(10, window=3, causal=False)


def test_cache_refuses_and_keeps_its_books():
    """What needs no kernel of PagedKVCache, on host tensors: pages that a window leaves behind, drafts that wait."""
    with pytest.raises(TypeError, match="dtype"):
        ssa_amd.PagedKVCache(4, 16, 2, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="sinks"):
        ssa_amd.PagedKVCache(4, 16, 2, 64, device="cpu", sinks=3)
    with pytest.raises(ValueError, match="window"):
        ssa_amd.PagedKVCache(4, 16, 2, 64, device="cpu", window=0)
    c = ssa_amd.PagedKVCache(20, 16, 2, 64, dtype=torch.int8, device="cpu", window=40, sinks=17)
    assert c.k_scales.shape == (20, 16, 2) and c.k_scales[0, :, 0].is_contiguous()
    s = c.add()
    c._pages[s], c._free = list(range(9)), list(range(9, 20))
    for length, behind in ((0, []), (70, []), (71, []), (87, [2]), (88, [2]), (103, [2, 3]), (143, [2, 3, 4, 5])):
        c._len[s] = length
        assert c._behind(s) == behind, length
        # the next token, at position `length`, sees none of their keys; the page after them it does
        for i in behind:
            assert all(x >= 17 and x <= length - 40 for x in range(16 * i, 16 * i + 16))
        nxt = (behind or [1])[-1] + 1
        assert any(x > length - 40 for x in range(16 * nxt, 16 * nxt + 16))
    c._gone[s].update([2, 3])
    assert c._behind(s) == [4, 5]
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="parents"):
        c.step(q, k, k, [s], [2], parents=[[-1]])
    with pytest.raises(ValueError, match="parents"):
        c.step(q, k, k, [s], [2], parents=[[-1, 1]])
    with pytest.raises(ValueError, match="64"):
        c.step(torch.zeros(65, 4, 64), None, None, [s], [65], parents=[list(range(-1, 64))])
    c._drafts[s] = 3
    with pytest.raises(ValueError, match="drafted"):
        c.step(q, k, k, [s], [2])
    for bad in ([0, 0], [2, 1], [3], [-1]):
        with pytest.raises(ValueError, match="ascend"):
            c.keep([s], [bad])
    with pytest.raises(ValueError, match="pair"):
        c.keep([s, s], [[0], [0]])
    c.keep([s], [[0, 1]])  # (a prefix moves nothing)
    assert c.length(s) == 142 and c._drafts[s] == 0
    free = c.free_pages
    c._drafts[s] = 20
    c.keep([s], [[]])
    assert c.length(s) == 122 and len(c._pages[s]) == 8 and c.free_pages == free + 1
    with pytest.raises(ValueError, match="given back"):
        c.read(s, 30, 60)
    with pytest.raises(ValueError, match="keys"):
        c.read(s, 60, 200)
    c.free(s)
    assert c.free_pages == 18  # (the two that the test marked as gone were never given back)
