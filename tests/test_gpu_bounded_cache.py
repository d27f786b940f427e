"""paged_step with windows, drafted trees and pages of 8 bits, paged_keep, paged_read and
PagedKVCache with them against the 64-bit oracle (tests/cache_oracle.py)."""

import math
import random

import pytest
import torch

from tests.cache_oracle import attend_set, held, sees, tree, values
from tests.dense_oracle import check

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4M3 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def bits(t):
    return t.contiguous().view(torch.uint8)


def batch(seed, dtype, seqs, h_q, h_kv, d, page, hold=None, window=0, sinks=0, trees=False, spare=2, behind=0):
    """Sequences (new, cached) with scattered pages; rows and keys of nobody hold NaN (codes of 8
    bits: NaN scales), and the table's entries of pages that no row sees are outside the pool."""
    g, r = torch.Generator().manual_seed(seed), random.Random(seed)
    counts = [-(-(m + c) // page) for m, c in seqs]
    pages = sum(counts) + spare
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), max(max(counts), 1) + 1), 10 ** 6, dtype=torch.int32)
    store = hold or dtype
    pools = {}
    for x in "kv":
        if hold:
            pools[x + "_pages"] = torch.randint(-128, 128, (pages, page, h_kv, d), generator=g).to(I8).view(hold)
            pools[x + "_scales"] = torch.full((pages, page, h_kv), math.nan)
        else:
            pools[x + "_pages"] = torch.full((pages, page, h_kv, d), math.nan, dtype=dtype)
    keys, at, parents = [], 0, []
    for b, (m, c) in enumerate(seqs):
        mine = perm[at:at + counts[b]]
        at += counts[b]
        up = tree(m, r) if trees else None
        parents.append(up)
        see = sees(m, c, up, window, sinks)[0].any(0)
        for i in range(counts[b]):
            # (new rows are written whether anybody sees them or not)
            if not window or see[i * page:(i + 1) * page].any() or (i + 1) * page > c:
                table[b, i] = mine[i]
        pair = []
        for x in "kv":
            rows = torch.randn(c + m, h_kv, d, generator=g).to(dtype)
            j = torch.arange(c)
            where = (mine[j // page], j % page)
            if hold:
                codes, scale = held(rows[:c], hold)
                pools[x + "_pages"].view(I8)[where] = codes.view(I8)
                pools[x + "_scales"][where] = scale
                pair.append(torch.cat([values(codes, scale), rows[c:].double()]))
            else:
                pools[x + "_pages"][where] = rows[:c]
                pair.append(rows)
        keys.append(pair)
    T = sum(m for m, _ in seqs)
    q = torch.randn(T + behind, h_q, d, generator=g).to(dtype)
    new = [torch.cat([x[i][c:].to(dtype) for x, (_, c) in zip(keys, seqs)] + [torch.full((behind, h_kv, d), math.nan, dtype=dtype)])
           for i in range(2)]
    starts = torch.tensor([sum(m for m, _ in seqs[:i]) for i in range(len(seqs) + 1)], dtype=torch.int32)
    s = dict(q=q, k=new[0], v=new[1], table=table, starts=starts,
             cached=torch.tensor([c for _, c in seqs], dtype=torch.int32), **pools)
    if trees:
        s["parents"] = torch.tensor([y for up in parents for y in up] + [-1] * behind, dtype=torch.int32)
    return s, keys, parents


def expect(s, keys, parents, seqs, cap=0.0, slopes=None, window=0, sinks=0):
    at = 0
    for b, (m, c) in enumerate(seqs):
        if m:
            see, qpos, kpos = sees(m, c, parents[b], window, sinks)
            yield b, at, m, attend_set(s["q"][at:at + m], *keys[b], see, qpos, kpos, cap, slopes)["out"]
        at += m


def pools_after(s, seqs, page, hold):
    """The pools with the new rows written."""
    want = {}
    for x in "kv":
        pages = s[x + "_pages"].clone()
        scales = s[x + "_scales"].clone() if hold else None
        at = 0
        for b, (m, c) in enumerate(seqs):
            j = torch.arange(c, c + m)
            where = (s["table"][b].long()[j // page], j % page)
            rows = s[x][at:at + m]
            if hold:
                codes, scale = held(rows, hold)
                pages.view(I8)[where] = codes.view(I8)
                scales[where] = scale
            else:
                pages[where] = rows
            at += m
        want[x + "_pages"] = pages
        if hold:
            want[x + "_scales"] = scales
    return want


CASES = [
    # dtype, pages of 8 bits, sequences (new, cached), tree, h_q, h_kv, d, page, window, sinks, cap, bias
    (F32, None, [(1, 0)], False, 2, 1, 8, 8, 1, 0, 0.0, False),
    (F32, None, [(1, 203)], False, 8, 2, 64, 16, 50, 4, 0.0, False),
    (BF16, None, [(1, 31), (1, 32), (1, 33), (1, 500), (0, 40), (1, 127)], False, 8, 2, 128, 8, 17, 9, 0.0, False),
    (BF16, None, [(1, 1000), (3, 77), (2, 1)], False, 28, 4, 128, 64, 300, 1, 4.0, True),
    (F32, None, [(2, 700), (1, 5)], False, 16, 1, 128, 32, 64, 40, 3.0, True),
    (BF16, None, [(5, 90), (6, 0), (8, 700)], False, 8, 2, 80, 8, 3, 2, 0.0, False),
    (BF16, None, [(1, 3000)], False, 16, 2, 64, 128, 1500, 130, 0.0, True),
    (BF16, None, [(70, 200)], False, 8, 2, 64, 16, 33, 4, 0.0, False),
    (BF16, None, [(150, 0)], False, 4, 4, 128, 32, 20, 70, 0.0, False),
    (F32, None, [(40, 100), (1, 64), (33, 0)], False, 6, 2, 96, 16, 37, 0, 2.0, False),
    (BF16, None, [(1, 600), (45, 2000), (0, 0), (1, 9), (130, 31)], False, 28, 4, 128, 32, 256, 4, 5.0, True),
    (BF16, None, [(300, 5000)], False, 16, 2, 128, 64, 2000, 100, 0.0, False),
    (F32, None, [(90, 900)], False, 4, 4, 128, 8, 70, 3, 0.0, True),
    # trees
    (F32, None, [(7, 203)], True, 8, 2, 64, 16, 0, 0, 0.0, False),
    (BF16, None, [(1, 0), (2, 5), (6, 31), (4, 300)], True, 8, 2, 128, 16, 0, 0, 0.0, True),
    (BF16, None, [(64, 500), (33, 64), (64, 0)], True, 16, 2, 64, 32, 0, 0, 0.0, False),
    (BF16, None, [(32, 1000), (31, 6), (1, 77)], True, 28, 4, 128, 64, 0, 0, 5.0, True),
    (F32, None, [(50, 130), (63, 1)], True, 6, 2, 96, 8, 0, 0, 2.0, True),
    (BF16, None, [(20, 4), (64, 700), (8, 0)], True, 8, 4, 128, 16, 5, 6, 0.0, True),
    (F32, None, [(13, 3), (6, 40)], True, 2, 1, 64, 8, 2, 5, 0.0, False),
    # 8 bits
    (F32, I8, [(1, 0)], False, 2, 1, 8, 8, 0, 0, 0.0, False),
    (F32, E4M3, [(1, 203)], False, 8, 2, 64, 16, 0, 0, 0.0, True),
    (BF16, I8, [(1, 31), (1, 32), (1, 33), (1, 500), (0, 40), (1, 127)], False, 8, 2, 128, 16, 0, 0, 0.0, False),
    (BF16, E4M3, [(1, 1000), (3, 77), (2, 1)], False, 28, 4, 128, 64, 0, 0, 4.0, True),
    (BF16, I8, [(5, 90), (6, 0), (8, 700)], False, 8, 2, 72, 8, 0, 0, 0.0, False),
    (BF16, E4M3, [(1, 3000)], False, 16, 2, 64, 128, 0, 0, 0.0, False),
    (F32, I8, [(2, 300), (1, 5)], False, 16, 1, 128, 32, 0, 0, 3.0, True),
    (BF16, I8, [(70, 200)], False, 8, 2, 64, 16, 0, 0, 0.0, False),
    (BF16, E4M3, [(150, 0), (40, 17)], False, 4, 4, 128, 32, 0, 0, 0.0, False),
    (F32, E4M3, [(40, 100), (1, 64), (33, 0)], False, 6, 2, 96, 16, 0, 0, 2.0, False),
    (F32, I8, [(90, 1000)], False, 4, 2, 120, 16, 0, 0, 0.0, False),
    (BF16, I8, [(200, 3000), (1, 64)], False, 16, 4, 128, 64, 0, 0, 0.0, True),
    # few rows over 8 bits, of every width, group and number of tokens
    (BF16, I8, [(1, 31), (1, 700)], False, 2, 1, 8, 8, 0, 0, 0.0, False),
    (BF16, E4M3, [(1, 100), (2, 1), (1, 33)], False, 4, 2, 24, 16, 0, 0, 0.0, True),
    (BF16, E4M3, [(1, 600), (1, 0)], False, 16, 1, 112, 32, 0, 0, 3.0, False),
    (BF16, I8, [(16, 505), (9, 100), (1, 64)], False, 2, 2, 128, 64, 0, 0, 0.0, False),
    (BF16, I8, [(7, 300), (8, 1030)], True, 4, 2, 80, 16, 0, 0, 0.0, True),
    (BF16, E4M3, [(16, 60), (16, 3), (11, 520)], True, 3, 3, 64, 8, 9, 5, 2000.0, True),
    (BF16, I8, [(1, 5000), (1, 40), (1, 900)], False, 14, 1, 128, 32, 300, 40, 0.0, True),
    (F32, I8, [(16, 505), (9, 100), (1, 64)], False, 2, 2, 128, 64, 0, 0, 0.0, False),
    # all together
    (BF16, I8, [(1, 600), (45, 2000), (0, 0), (1, 9), (130, 31)], False, 28, 4, 128, 32, 256, 4, 5.0, True),
    (BF16, E4M3, [(20, 4), (64, 700), (8, 0)], True, 8, 4, 128, 16, 5, 6, 0.0, True),
    (F32, I8, [(7, 203), (5, 1)], True, 8, 2, 64, 16, 30, 2, 0.0, True),
    (F32, E4M3, [(64, 333)], True, 12, 4, 128, 64, 100, 64, 1.5, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_step(dev, case):
    from ssa_amd import paged_read, paged_step

    dtype, hold, seqs, trees, h_q, h_kv, d, page, window, sinks, cap, bias = case
    print(f"bounded {case}", flush=True)
    slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)]) if bias else None
    s, keys, parents = batch(51, dtype, seqs, h_q, h_kv, d, page, hold, window, sinks, trees, behind=3)
    x = {n: t.to(dev) for n, t in s.items()}
    out = torch.full(x["q"].shape, 7.0, device=dev, dtype=dtype)
    kw = dict(softcap=cap or None, slopes=None if slopes is None else slopes.to(dev), check=True)
    if window:
        kw.update(window=window, sinks=sinks)
    assert paged_step(**x, out=out, **kw) is out
    T = int(s["starts"][-1])
    assert (out[T:] == 7).all(), "rows behind the last sequence"
    rule = dict(cap=cap, slopes=slopes, window=window, sinks=sinks)
    for b, at, m, (value, bound) in expect(s, keys, parents, seqs, **rule):
        check(out[at:at + m], value, bound, f"sequence {b}")
    # the pools hold the new rows, and nothing else of them changed
    for name, want in pools_after(s, seqs, page, hold).items():
        assert torch.equal(bits(x[name].cpu()), bits(want)), name
    # read back; and where the keys are there now, the same without k and v and with tight bounds
    part = {n: x[n] for n in ("k_pages", "v_pages", "table", "starts")}
    scales = {n: x[n] for n in ("k_scales", "v_scales") if hold}
    back = paged_read(**part, first=x["cached"], tokens=T + 3, dtype=F32 if hold else None, check=True, **scales)
    at = 0
    for b, (m, c) in enumerate(seqs):
        for i, got in enumerate(back):
            rows = s["kv"[i]][at:at + m]
            want = values(*held(rows, hold)).float() if hold else rows
            assert torch.equal(got[at:at + m].cpu(), want)
            if hold:
                keys[b][i][c:] = values(*held(rows, hold))
        at += m
    assert not back[0][T:].any() and not back[1][T:].any()
    x["k"] = x["v"] = None
    again = paged_step(**x, max_new=max(max(m for m, _ in seqs), 1), max_len=max(m + c for m, c in seqs), **kw)
    for b, at, m, (value, bound) in expect(s, keys, parents, seqs, **rule):
        check(again[at:at + m], value, bound, f"sequence {b} without append")
    assert not again[T:].any()


def test_a_chain_is_a_tree(dev):
    """Parents of a chain give what no parents give, and a window that reaches every key none."""
    from ssa_amd import paged_step

    seqs = [(9, 100), (1, 40), (17, 0)]
    for dtype, hold in ((BF16, None), (F32, None), (BF16, I8)):
        s, keys, _ = batch(52, dtype, seqs, 8, 2, 64, 16, hold)
        up = torch.cat([torch.arange(-1, m - 1) for m, _ in seqs]).to(torch.int32)
        x = {n: t.to(dev) for n, t in s.items()}
        a = paged_step(**{**x, "parents": up.to(dev)}, check=True)
        for got in (a, paged_step(**x, window=118, sinks=3), paged_step(**x, window=1 << 40)):
            for b, at, m, (value, bound) in expect(s, keys, [None] * 3, seqs):
                check(got[at:at + m], value, bound, f"sequence {b}")


@pytest.mark.parametrize("hold", [None, I8, E4M3])
def test_values_that_are_not_finite(dev, hold):
    """A NaN or an infinity that a row sees reaches it; one that it does not see (behind its window,
    on another branch of the tree) has no influence, in few rows and many."""
    from ssa_amd import paged_step

    for dtype in (F32, BF16):
        for m, trees, window in ((1, False, 60), (6, True, 0), (40, False, 25), (60, True, 0), (50, True, 20)):
            seqs = [(m, 150)]
            print(f"not finite {hold} {dtype} {m} {trees} {window}", flush=True)
            s, keys, parents = batch(53, dtype, seqs, 4, 2, 64, 16, hold, window, 2 if window else 0, trees)
            see, qpos, kpos = sees(m, 150, parents[0], window, 2 if window else 0)
            # every key that some row does not see and another does, and one that none sees
            bad = [int(j) for j in ((~see).any(0) & see.any(0)).nonzero()[:, 0][::7]] or [0]
            for j in bad[:3] + ([int((~see.any(0)).nonzero()[0])] if (~see.any(0)).any() else []):
                x = {n: t.clone() for n, t in s.items()}
                if j >= 150:
                    x["v"][j - 150, 0, 9] = math.inf
                    x["k"][j - 150, 1, 3] = math.nan
                elif int(s["table"][0, j // 16]) < 10 ** 6:
                    pg = s["table"][0, j // 16]
                    if hold:
                        x["v_scales"][pg, j % 16, 0] = math.nan
                        x["k_scales"][pg, j % 16, 1] = math.nan
                    else:
                        x["v_pages"][pg, j % 16, 0, 9] = math.inf
                        x["k_pages"][pg, j % 16, 1, 3] = math.nan
                out = paged_step(**{n: t.to(dev) for n, t in x.items()}, window=window or None,
                                 sinks=2 if window else 0).cpu()
                hit = see[:, j]
                (_, _, _, (value, bound)), = expect(s, keys, parents, seqs, window=window, sinks=2 if window else 0)
                if not hit.all():
                    check(out[~hit], value[~hit], bound[~hit], f"rows that do not see key {j}")
                if j >= 150 or int(s["table"][0, j // 16]) < 10 ** 6:
                    assert torch.isnan(out[hit][:, 2:]).all(), "a key that is NaN"
                    assert not torch.isfinite(out[hit][:, :2, 9]).any()


def test_pages_of_nothing_but_masked_keys_are_not_read(dev):
    """Entries between the first keys and the window may hold anything: check=True finds no fault
    (batch puts them outside the pool), through one launch and through parts."""
    from ssa_amd import paged_step

    for seqs, window in (([(1, 4000)], 40), ([(1, 4000), (2, 3000)], 1500), ([(100, 4000)], 70), ([(20, 4000), (5, 900)], 8)):
        for hold in (None, I8):
            s, keys, parents = batch(54, BF16, seqs, 8, 2, 128, 8, hold, window, 11)
            assert (s["table"][0, 2:300] == 10 ** 6).any()
            out = paged_step(**{n: t.to(dev) for n, t in s.items()}, window=window, sinks=11, check=True)
            for b, at, m, (value, bound) in expect(s, keys, parents, seqs, window=window, sinks=11):
                check(out[at:at + m], value, bound, f"sequence {b}")


def test_bad_parents_and_sequences(dev):
    from ssa_amd import paged_step

    seqs = [(5, 40), (6, 30), (5, 20)]
    for hold in (None, I8):
        s, keys, parents = batch(55, BF16, seqs, 4, 2, 64, 16, hold, trees=True)
        for bad, at in ((4, 3), (-2, 7), (1 << 30, 12), (-(1 << 31), 5)):
            x = {n: t.to(dev) for n, t in s.items()}
            x["parents"][at] = bad
            out = paged_step(**x)
            ups = [list(p) for p in parents]
            b = 0 if at < 5 else 1 if at < 11 else 2
            ups[b][at - (0, 5, 11)[b]] = -1
            for b, a, m, (value, bound) in expect(s, keys, ups, seqs):
                check(out[a:a + m], value, bound, f"sequence {b}")
            with pytest.raises(IndexError):
                paged_step(**x, check=True)
        # a sequence with more drafts than the bound is left out, the others are not
        x = {n: t.to(dev) for n, t in s.items()}
        out = paged_step(**x, max_new=5)
        assert not out[5:11].any()
        for b, a, m, (value, bound) in expect(s, keys, parents, seqs):
            if b != 1:
                check(out[a:a + m], value, bound, f"sequence {b}")


@pytest.mark.parametrize("hold", [I8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rounding_of_held_rows(dev, dtype, hold):
    """Codes next to the borders between two, rows of one value, of zeros, tiny, huge and not finite:
    the nearest code of the exact quotient, bit by bit."""
    from ssa_amd import paged_read, paged_step

    g = torch.Generator().manual_seed(56)
    d, h_kv, page = 128, 2, 16
    rows = torch.randn(400, h_kv, d, generator=g, dtype=torch.float64)
    most = 127.0 if hold == I8 else 448.0
    # multiples of half a code (ties), and floats beside them
    half = torch.randint(-253, 254, (200, h_kv, d), generator=g).double() / 2
    half[..., 0] = most
    if hold == E4M3:
        grid = torch.arange(256, dtype=torch.uint8).view(E4M3).float().double()
        grid = grid[torch.isfinite(grid)].sort().values
        mid = (grid[1:] + grid[:-1]) / 2
        half = mid[torch.randint(0, len(mid), (200, h_kv, d), generator=g)]
        half[..., 0] = most
    unit = torch.exp2(torch.randint(-20, 20, (200, 1, 1), generator=g).double())
    unit[100:] *= 1.0 + torch.rand(100, 1, 1, generator=g, dtype=torch.float64)
    near = (half * unit).float()
    near[50:] = torch.nextafter(near[50:], torch.where(torch.rand(near[50:].shape, generator=g) < 0.5, -1.0, 1.0) * 1e30)
    rows[:200] = near.double()
    rows[200], rows[201], rows[202], rows[203] = 0.0, 2.0 ** -101, 2.0 ** -99, 3e38
    rows[204, 0, 5], rows[205, 1, 0], rows[206, 0, 127] = math.nan, math.inf, -math.inf
    rows[207], rows[208] = -1.0, 1e-40
    rows = rows.to(dtype)
    T = len(rows)
    pages = -(-T // page)
    x = dict(k_pages=torch.zeros(pages, page, h_kv, d, device=dev, dtype=I8).view(hold),
             v_pages=torch.zeros(pages, page, h_kv, d, device=dev, dtype=I8).view(hold),
             k_scales=torch.zeros(pages, page, h_kv, device=dev), v_scales=torch.zeros(pages, page, h_kv, device=dev),
             table=torch.arange(pages, device=dev, dtype=torch.int32)[None],
             starts=torch.tensor([0, T], device=dev, dtype=torch.int32))
    zero = torch.zeros(1, device=dev, dtype=torch.int32)
    k = rows.to(dev)
    paged_step(torch.zeros(T, 2, d, device=dev, dtype=dtype), k, k.flip(-1), cached=zero, **x)
    codes, scale = held(rows, hold)
    for name, want, sc in (("k", codes, scale), ("v", codes.view(I8).flip(-1).view(hold), scale)):
        got = x[name + "_pages"].view(-1, h_kv, d)[:T].cpu()
        assert torch.equal(torch.nan_to_num(x[name + "_scales"].view(-1, h_kv)[:T].cpu(), nan=-1.0), torch.nan_to_num(sc, nan=-1.0))
        # (zeros of either sign stand for the same)
        assert torch.equal(got.float(), want.float()), name
    for out in (F32, BF16):
        back, _ = paged_read(first=zero, tokens=T, dtype=out, **x)
        want = values(codes, scale).float().to(out)
        assert torch.equal(torch.nan_to_num(back.cpu(), nan=-7.0), torch.nan_to_num(want, nan=-7.0))


def test_every_code(dev):
    """All 256 codes of both kinds, as keys' values and read back."""
    from ssa_amd import paged_read, paged_step

    for hold in (I8, E4M3):
        codes = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(I8)
        if hold == E4M3:
            codes = codes[torch.isfinite(codes.view(E4M3).float())]
        n, d, page = len(codes), 8, 8
        pool = torch.zeros(-(-n // page), page, 1, d, dtype=I8)
        pool.view(-1, d)[:n] = codes[:, None]
        scales = torch.full(pool.shape[:3], 0.37)
        x = dict(k_pages=torch.zeros_like(pool).view(hold), v_pages=pool.view(hold), k_scales=torch.ones_like(scales),
                 v_scales=scales, table=torch.arange(len(pool), dtype=torch.int32)[None],
                 starts=torch.tensor([0, 1], dtype=torch.int32))
        x = {a: t.to(dev) for a, t in x.items()}
        want = codes.view(hold).float() * torch.tensor(0.37)
        for dtype in (F32, BF16):
            # with a window of one, each key by itself
            for i in range(0, n, 5):
                at = torch.tensor([i], device=dev, dtype=torch.int32)
                out = paged_step(torch.zeros(1, 1, d, device=dev, dtype=dtype), None, None, cached=at, window=1, **x)
                r = 2.0 ** -23 if dtype == F32 else 2.0 ** -7
                assert ((out[0, 0].cpu().float() - want[i]).abs() <= r * want[i].abs()).all()
        back = paged_read(first=torch.zeros(1, device=dev, dtype=torch.int32), tokens=n,
                          **{**x, "starts": torch.tensor([0, n], device=dev, dtype=torch.int32)}, dtype=F32)[1]
        assert torch.equal(back[:, 0, 0].cpu(), want)


@pytest.mark.parametrize("hold", [None, I8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_keep(dev, dtype, hold):
    from ssa_amd import paged_keep

    for seed, (page, d, h_kv, top) in enumerate([(8, 64, 2, 64), (16, 128, 3, 20), (64, 8, 1, 5), (16, 72, 2, 1)]):
        r = random.Random(seed)
        seqs = [(m, r.randrange(0, 90)) for m in (64, 1, 20, 33, 7)]
        s, _, _ = batch(60 + seed, dtype, seqs, h_kv, h_kv, d, page, hold, trees=True)
        kept = []
        for m, _ in seqs:
            n = r.randrange(0, min(m, top) + 1)
            kept.append(sorted(r.sample(range(m), n)) + [-1] * (top - n))
        kept[3] = (list(range(min(33, top))) + [-1] * top)[:top]
        want = pools_after(s, seqs, page, hold)
        x = {n: t.to(dev) for n, t in {**s, **want}.items()}
        scales = {n: x[n] for n in ("k_scales", "v_scales") if hold}
        paged_keep(x["k_pages"], x["v_pages"], x["table"], x["cached"], torch.tensor(kept, device=dev, dtype=torch.int32),
                   check=True, **scales)
        for name, t in want.items():
            old = t.clone()
            for b, (m, c) in enumerate(seqs):
                for i, j in enumerate(y for y in kept[b] if y >= 0):
                    a, z = c + i, c + j
                    src, dst = (s["table"][b].long()[z // page], z % page), (s["table"][b].long()[a // page], a % page)
                    t[dst] = old[src]
            assert torch.equal(bits(x[name].cpu()), bits(t)), name
    # a list that does not ascend ends there, one past the table too
    for bad, good in (([0, 2, 2, 5], 2), ([3, 1, 5, 6], 1), ([0, 2, 1 << 30, (1 << 30) + 1], 2)):
        x = {n: t.to(dev) for n, t in {**s, **want}.items()}
        scales = {n: x[n] for n in ("k_scales", "v_scales") if hold}
        rows = torch.tensor([bad] + [[-1] * 4] * 4, device=dev, dtype=torch.int32)
        args = (x["k_pages"], x["v_pages"], x["table"], x["cached"])
        with pytest.raises(IndexError):
            paged_keep(*args, rows, check=True, **scales)
        t, c, page = want["k_pages"].clone(), seqs[0][1], 16
        for i, j in enumerate(bad[:good]):
            t[s["table"][0].long()[(c + i) // page], (c + i) % page] = want["k_pages"][s["table"][0].long()[(c + j) // page], (c + j) % page]
        assert torch.equal(bits(x["k_pages"].cpu()), bits(t))


def test_strided_pools(dev):
    """K and V in one pool, heads before tokens, scales in any order; rows of q, k, v and out inside others."""
    from ssa_amd import paged_keep, paged_read, paged_step

    seqs = [(20, 77), (1, 300), (3, 9)]
    for dtype, hold in ((BF16, None), (BF16, I8), (F32, E4M3)):
        s, keys, parents = batch(57, dtype, seqs, 8, 2, 64, 16, hold, trees=True)
        pages, page, h, d = s["k_pages"].shape
        x = {n: t.to(dev) for n, t in s.items()}
        one = torch.zeros(pages, 2, h, page, d + 16, device=dev, dtype=I8 if hold else dtype)
        kv = [one[:, i, :, :, :d].transpose(1, 2) for i in range(2)]
        for i, n in enumerate(("k_pages", "v_pages")):
            kv[i].copy_(x[n].view(I8) if hold else x[n])
            x[n] = kv[i].view(hold) if hold else kv[i]
        if hold:
            both = torch.zeros(h, pages, page, 2, device=dev)
            for i, n in enumerate(("k_scales", "v_scales")):
                both[..., i].copy_(x[n].permute(2, 0, 1))
                x[n] = both[..., i].permute(1, 2, 0)
        wide = torch.zeros(len(x["q"]), 16, d + 8, device=dev, dtype=dtype)
        wide[:, 4:12, :d] = x["q"]
        x["q"] = wide[:, 4:12, :d]
        out = torch.zeros(len(wide), 8, d + 8, device=dev, dtype=dtype)[..., :d]
        paged_step(**x, out=out, window=60, sinks=3, check=True)
        for b, at, m, (value, bound) in expect(s, keys, parents, seqs, window=60, sinks=3):
            check(out[at:at + m], value, bound, f"sequence {b}")
        want = pools_after(s, seqs, page, hold)
        for n, t in want.items():
            assert torch.equal(bits(x[n].cpu()), bits(t)), n
        assert not one[..., d:].any(), "between the rows"
        scales = {n: x[n] for n in ("k_scales", "v_scales") if hold}
        kept = torch.tensor([[1, 4, 19], [-1] * 3, [0, 2, -1]], device=dev, dtype=torch.int32)
        paged_keep(x["k_pages"], x["v_pages"], x["table"], x["cached"], kept, check=True, **scales)
        k, v = paged_read(x["k_pages"], x["v_pages"], x["table"], x["starts"], x["cached"], 24, check=True, **scales)
        for got, name in ((k, "k"), (v, "v")):
            rows = s[name]
            for at, src in ((0, 1), (1, 4), (2, 19), (3, 3), (20, 20), (21, 21), (22, 23)):
                ref = values(*held(rows[src], hold)).float().to(BF16) if hold else rows[src]
                assert torch.equal(got[at].cpu(), ref), (name, at)


def test_captured_and_on_streams(dev):
    """A captured tree step over 8 bits with its keep follows what it reads; eager calls on two streams agree."""
    from ssa_amd import paged_keep, paged_step

    seqs = [(9, 900), (4, 250), (12, 64)]
    for hold, window in ((None, 200), (I8, 0), (E4M3, 300)):
        s, _, _ = batch(58, BF16, seqs, 8, 2, 128, 16, hold, trees=True)
        x = {n: t.to(dev) for n, t in s.items()}
        scales = {n: x[n] for n in ("k_scales", "v_scales") if hold}
        kept = torch.tensor([[0, 3, 7], [1, 2, -1], [5, 6, 11]], device=dev, dtype=torch.int32)
        kw = dict(max_new=12, max_len=1000, window=window or None, sinks=4 if window else 0)

        def step():
            out = paged_step(**x, **kw)
            paged_keep(x["k_pages"], x["v_pages"], x["table"], x["cached"], kept, **scales)
            return out

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for turn in range(4):
            x["q"].add_(0.25)
            x["k"].mul_(0.9)
            if turn:
                x["cached"].sub_(7)
                x["parents"][6] = turn
                kept[0, 1] = 3 + turn % 3
            start = {n: x[n].clone() for n in ("k_pages", "v_pages", *scales)}
            graph.replay()
            torch.cuda.synchronize()
            after = {n: bits(x[n]).clone() for n in start}
            for n, t in start.items():
                x[n].view(torch.uint8).copy_(t.view(torch.uint8))
            eager = step()
            assert torch.equal(out, eager)
            assert all(torch.equal(after[n], bits(x[n])) for n in start)
        quiet = {**x, "k": None, "v": None}
        want = paged_step(**quiet, **kw)
        torch.cuda.synchronize()
        got = []
        for st in [torch.cuda.Stream() for _ in range(2)] * 3:
            with torch.cuda.stream(st):
                got.append(paged_step(**quiet, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_far_pages(dev):
    """Codes past 2^31 of the pool's elements and 2^32 of its bytes."""
    from ssa_amd import paged_keep, paged_read, paged_step

    page, h_kv, d = 64, 8, 128
    pages = (1 << 32) // (page * h_kv * d) + 40
    big = {n: torch.zeros(pages, page, h_kv, d, device=dev, dtype=I8) for n in ("k_pages", "v_pages")}
    big.update({n: torch.zeros(pages, page, h_kv, device=dev) for n in ("k_scales", "v_scales")})
    seqs = [(3, 300), (30, 100)]
    s, keys, parents = batch(59, BF16, seqs, 8, h_kv, d, page, I8, trees=True)
    small = s["k_pages"].shape[0]
    for n, t in big.items():
        t[pages - small:] = s[n].to(dev)
    s["table"] = torch.where(s["table"] < small, s["table"] + pages - small, s["table"])
    x = {n: t.to(dev) for n, t in s.items()}
    x.update(big)
    out = paged_step(**x, check=True)
    for b, at, m, (value, bound) in expect(s, keys, parents, seqs):
        check(out[at:at + m], value, bound, f"sequence {b}")
    kept = torch.tensor([[0, 2], [5, 29]], device=dev, dtype=torch.int32)
    scales = {n: x[n] for n in ("k_scales", "v_scales")}
    paged_keep(x["k_pages"], x["v_pages"], x["table"], x["cached"], kept, check=True, **scales)
    k, _ = paged_read(x["k_pages"], x["v_pages"], x["table"], x["starts"], x["cached"], 33, dtype=F32, check=True, **scales)
    for at, src in ((0, 0), (1, 2), (3, 8), (4, 32)):
        assert torch.equal(k[at].cpu(), values(*held(s["k"][src], I8)).float())


def test_long_positions(dev):
    """A window at the end of a sequence of nearly 2^31 keys: only its pages and the first ones exist."""
    from ssa_amd import paged_step

    page, width = 4096, (1 << 31) // 4096 - 1
    cached = width * page - 40
    g = torch.Generator().manual_seed(61)
    for m, hold in ((1, None), (33, None), (5, I8)):
        pool = [torch.randn(3, page, 2, 64, generator=g).to(BF16) for _ in range(2)]
        table = torch.full((1, width), 10 ** 6, dtype=torch.int32)
        table[0, 0], table[0, width - 1], table[0, width - 2] = 0, 1, 2
        window, sinks = page, 5
        rows = [torch.randn(m, 2, 64, generator=g).to(BF16) for _ in range(2)]
        x = dict(table=table, starts=torch.tensor([0, m], dtype=torch.int32), cached=torch.tensor([cached], dtype=torch.int32),
                 q=torch.randn(m, 4, 64, generator=g).to(BF16), k=rows[0], v=rows[1])
        seen = []
        for i, n in enumerate("kv"):
            codes, scale = held(pool[i], I8) if hold else (pool[i], None)
            x[n + "_pages"] = codes
            if hold:
                x[n + "_scales"] = scale
            full = values(codes, scale) if hold else codes.double()
            seen.append(torch.cat([full[0, :sinks], full[2], full[1, :page - 40], rows[i].double()]))
        kpos = torch.cat([torch.arange(sinks), torch.arange((width - 2) * page, cached + m)])
        qpos = cached + torch.arange(m)
        see = (kpos[None] <= qpos[:, None]) & ((qpos[:, None] - kpos[None] < window) | (kpos[None] < sinks))
        out = paged_step(**{n: t.to(dev) for n, t in x.items()}, window=window, sinks=sinks, check=True)
        check(out, *attend_set(x["q"], *seen, see, qpos, kpos)["out"], f"{m} {hold}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hold,window,sinks", [(None, 40, 4), (I8, None, 0), (E4M3, 70, 20), (None, None, 0)])
def test_cache(dev, dtype, hold, window, sinks):
    """Prompts in chunks, single tokens, drafted trees with what is kept of them, sequences that come and go:
    every output against the whole sequence's rows, and the pages that a window leaves behind go back."""
    from ssa_amd import PagedKVCache

    r, g = random.Random(3), torch.Generator().manual_seed(62)
    h_q, h_kv, d, page = 8, 2, 64, 16
    cache = PagedKVCache(60, page, h_kv, d, dtype=hold or dtype, window=window, sinks=sinks)
    rows = {}  # sequence -> (k, v) as they are given, in 64 bits as they are held
    def draw(m):
        return [torch.randn(m, h, d, generator=g).to(dtype) for h in (h_q, h_kv, h_kv)]

    def as_held(t):
        return values(*held(t, hold)) if hold else t.double()

    for turn in range(14):
        if turn in (0, 3):
            s = cache.add()
            rows[s] = [torch.zeros(0, h_kv, d, dtype=torch.float64) for _ in range(2)]
        if turn == 9:
            gone = next(iter(rows))
            del rows[gone]
            cache.free(gone)
        seqs = list(rows)
        trees = turn % 3 == 2
        counts = [r.randrange(1, 30) if trees else r.choice([1, 1, 37, 90]) for _ in seqs]
        ups = [tree(m, r) for m in counts] if trees else None
        new = [draw(m) for m in counts]
        q, k, v = (torch.cat([x[i] for x in new]).to(dev) for i in range(3))
        print(f"cache turn {turn} {counts} {trees}", flush=True)
        out = cache.step(q, k, v, seqs, counts, parents=ups)
        at = 0
        for i, s in enumerate(seqs):
            c, m = len(rows[s][0]), counts[i]
            see, qpos, kpos = sees(m, c, ups[i] if trees else None, window or 0, sinks)
            full = [torch.cat([a, b.double()]) for a, b in zip(rows[s], new[i][1:])]
            check(out[at:at + m], *attend_set(new[i][0], *full, see, qpos, kpos)["out"], f"turn {turn} sequence {s}")
            at += m
        kept = []
        for i, s in enumerate(seqs):
            keep = list(range(counts[i]))
            if trees:
                keep, x = [], r.randrange(-1, counts[i])
                while x >= 0:
                    keep.insert(0, x)
                    x = ups[i][x]
            kept.append(keep)
            rows[s] = [torch.cat([a, as_held(b)[keep]]) for a, b in zip(rows[s], new[i][1:])]
        if trees:
            with pytest.raises(ValueError, match="drafted"):
                cache.step(q[:1], k[:1], v[:1], seqs[:1], [1])
            cache.keep(seqs, kept)
        for s in seqs:
            assert cache.length(s) == len(rows[s][0])
            first = max(0, cache.length(s) - (window or cache.length(s)))
            for got, want in zip(cache.read(s, first, dtype=torch.float32 if hold else None), rows[s]):
                assert torch.equal(got.cpu().double(), want[first:].float().double())
    if window:
        s = max(rows, key=lambda x: len(rows[x][0]))
        n = cache.length(s)
        live = [i for i in range(len(cache._pages[s])) if i not in cache._gone[s]]
        assert n > window + 100 and len(live) <= (window + 90 + sinks) // page + 4
        with pytest.raises(ValueError, match="given back"):
            cache.read(s)
    for s in list(rows):
        cache.free(s)
    assert cache.free_pages == 60


@pytest.mark.parametrize("hold", [I8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_own_rows_across_parts(dev, dtype, hold):
    """New tokens on both sides of a border between parts, with hidden keys in the window's first tile whose
    codes stand for NaN: the rows that are computed again count every key once."""
    from ssa_amd import paged_step

    for m, window in ((14, 300), (3, 290), (16, 520)):
        for cached in range(560, 660, 4):
            s, keys, parents = batch(63, dtype, [(m, cached)], 2, 2, 64, 8, hold, window, 0)
            x = {n: t.clone() for n, t in s.items()}
            lo = cached + 1 - window
            for j in range(lo // 8 * 8, lo):   # (of the page that holds the window's first key)
                x["v_scales"][x["table"][0, j // 8], j % 8] = math.nan
            out = paged_step(**{n: t.to(dev) for n, t in x.items()}, window=window, check=True)
            (_, _, _, (value, bound)), = expect(s, keys, parents, [(m, cached)], window=window)
            check(out, value, bound, f"{m} {window} {cached}")


@pytest.mark.parametrize("hold", [None, I8, E4M3])
@pytest.mark.parametrize("dtype,h_q,m,trees", [(BF16, 2, 1, False), (F32, 2, 3, False), (BF16, 8, 9, False), (F32, 4, 30, True), (BF16, 1, 16, True)])
def test_windows_that_leave_no_cached_key(dev, dtype, hold, h_q, m, trees):
    """A window of one key: no page of the cached keys is looked up, wherever the new ones begin."""
    seqs = [(m, 128), (1, 32), (m, 40), (m, 0), (1, 56), (0, 64), (2, 127)]
    for sinks in (0, 1):
        test_step(dev, (dtype, hold, seqs, trees, h_q, 1, 64, 8, 1, sinks, 0.0, False))


@pytest.mark.parametrize("dtype,m,g", [(BF16, 1, 4), (BF16, 9, 2), (F32, 1, 4), (BF16, 30, 1), (BF16, 40, 4)])
def test_rows_without_a_key_are_not_looked_at(dev, dtype, m, g):
    """Pages of e4m3 whose other rows hold codes for NaN take no longer than pages of zeros (the rows
    that such a code reached would be computed again, key by key)."""
    from ssa_amd import paged_step

    seqs, h_kv = [(m, 4001)] * 4, 2
    s, _, _ = batch(64, dtype, seqs, h_kv * g, h_kv, 128, 64, E4M3)
    x = {n: t.to(dev) for n, t in s.items()}
    took = []
    for fill in (0, 0x7F):
        y = {n: t.clone() for n, t in x.items()}
        for n in ("k_pages", "v_pages"):
            flat = y[n].view(I8)
            for b in range(4):
                last = int(s["table"][b, 4001 // 64])
                flat[last, 4001 % 64:] = fill
        for keys_there in (False, True):
            if keys_there:
                y["k"] = y["v"] = None  # (the pages hold them now)
            z = dict(y, max_new=m, max_len=4001 + m)
            for _ in range(3):
                paged_step(**z)
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            best = 1e9
            for _ in range(5):
                a.record()
                for _ in range(10):
                    paged_step(**z)
                b.record()
                b.synchronize()
                best = min(best, a.elapsed_time(b))
            took.append(best)
    assert took[2] < 3 * took[0] and took[3] < 3 * took[1], took


def test_rows_aligned_to_8_bytes(dev):
    """Codes whose rows lie at odd multiples of 8 bytes."""
    from ssa_amd import paged_keep, paged_read, paged_step

    for dtype, m in ((BF16, 1), (BF16, 12), (BF16, 40), (F32, 3)):
        seqs = [(m, 300), (1, 70)]
        s, keys, parents = batch(65, dtype, seqs, 8, 2, 64, 16, I8)
        x = {n: t.to(dev) for n, t in s.items()}
        pages, page, h, d = x["k_pages"].shape
        for i, n in enumerate(("k_pages", "v_pages")):
            wide = torch.zeros(pages * page * h * (d + 8) + 8, device=dev, dtype=I8)[8:].view(pages, page, h, d + 8)
            wide[..., :d] = x[n]
            x[n] = wide[..., :d]
        out = paged_step(**x, check=True)
        for b, at, n, (value, bound) in expect(s, keys, parents, seqs):
            check(out[at:at + n], value, bound, f"sequence {b}")
        kept = torch.tensor([[0, 2] if m > 2 else [0, -1], [0, -1]], device=dev, dtype=torch.int32)
        scales = {n: x[n] for n in ("k_scales", "v_scales")}
        paged_keep(x["k_pages"], x["v_pages"], x["table"], x["cached"], kept, check=True, **scales)
        k, _ = paged_read(x["k_pages"], x["v_pages"], x["table"], x["starts"], x["cached"], m + 1, dtype=F32, check=True, **scales)
        want = s["k"][[0, 2] if m > 2 else [0]]
        assert torch.equal(k[:len(want)].cpu(), values(*held(want, I8)).float())
