"""paged_read's rounding and what rows without a key hold, bit by bit."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4M3 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def nearest_bf16(x):
    """float64 to bfloat16 in one rounding, ties to even (torch goes by way of float32): for a value between
    2^e and 2^(e + 1) a multiple of 2^(e - 7), of 2^-133 below the smallest normal one."""
    e = torch.frexp(x)[1].double().clamp(min=-125) - 1  # (frexp: a value in [0.5, 1) times 2^e)
    step = torch.exp2(e - 7)
    y = (x / step).round() * step
    return torch.where(torch.isfinite(x), y, x).float().to(BF16)


def test_nearest_bf16():
    """The reference itself, on the host's grid of values: what a bfloat16 holds stays, ties go to even."""
    grid = torch.arange(0, 0x7F80, dtype=torch.int16).view(BF16).double()
    assert torch.equal(nearest_bf16(grid).double(), grid)
    mid = (grid[1:] + grid[:-1]) / 2
    even = torch.where(torch.arange(len(mid)) % 2 == 0, grid[:-1], grid[1:])
    assert torch.equal(nearest_bf16(mid).double(), even)
    for way in (grid[1:], grid[:-1]):
        assert torch.equal(nearest_bf16(torch.nextafter(mid, way)).double(), way)


@pytest.mark.parametrize("hold", [I8, E4M3])
def test_codes_are_read_in_one_rounding(dev, hold):
    from ssa_amd import paged_read

    g = torch.Generator().manual_seed(81)
    T, h, d, page = 4096, 2, 128, 16
    codes = torch.randint(-128, 128, (2, T, h, d), generator=g).to(I8)
    if hold == E4M3:
        codes = torch.where(codes.view(E4M3).float().isnan(), 3, codes)
    scales = torch.exp2(torch.rand(2, T, h, generator=g) * 12 - 9)
    scales[:, 0] = 0.022805606946349144
    codes[:, 0, :, 0] = 17
    scales[:, 1], scales[:, 2], scales[:, 3], scales[:, 4], scales[:, 5] = 2.0 ** -126, 1.3e-42, 3.1e36, math.nan, 0.0
    scales[:, 6:200] = torch.exp2(torch.rand(2, 194, h, generator=g) * 60 - 149)  # (products around 2^-100 and below fp32's)
    scales[:, 200] = -scales[:, 201]
    pools = [x.view(hold).view(-1, page, h, d).to(dev) for x in codes]
    both = [x.view(-1, page, h).to(dev) for x in scales]
    at = dict(table=torch.arange(T // page, device=dev, dtype=torch.int32)[None],
              starts=torch.tensor([0, T], device=dev, dtype=torch.int32), first=torch.zeros(1, device=dev, dtype=torch.int32))
    exact = codes.view(hold).float().double() * scales.double()[..., None]
    for dtype, want in ((BF16, nearest_bf16(exact)), (F32, exact.float())):
        got = paged_read(*pools, tokens=T, dtype=dtype, k_scales=both[0], v_scales=both[1], check=True, **at)
        for x, y in zip(got, want):
            x = x.cpu()
            assert torch.equal(x.isnan(), y.isnan()) and torch.equal(torch.nan_to_num(x, nan=0.0), torch.nan_to_num(y, nan=0.0))
    if hold == I8:
        assert float(exact[0, 0, 0, 0]) == 17 * float(torch.tensor(0.022805606946349144))
        assert float(nearest_bf16(exact)[0, 0, 0, 0]) == 0.388671875
    assert not torch.equal(torch.nan_to_num(nearest_bf16(exact)), torch.nan_to_num(exact.float().to(BF16))), "no product tells them apart"


@pytest.mark.parametrize("dtype,m,g", [(BF16, 1, 4), (BF16, 9, 2), (F32, 1, 4), (BF16, 30, 1), (BF16, 40, 4), (F32, 40, 2)])
@pytest.mark.parametrize("cached", [13, 4001])
def test_codes_of_rows_without_a_key_change_no_bit(dev, dtype, m, g, cached):
    """Pages of e4m3 whose rows behind the last key hold codes for NaN give the bits that zeros there give: a
    row that one of them reached would be computed again key by key, in another order of its sums."""
    from ssa_amd import paged_step
    from tests.cache_oracle import attend_set, held, sees, values
    from tests.dense_oracle import check
    from tests.test_gpu_bounded_cache import batch

    seqs, h_kv, page = [(m, cached)] * 4, 2, 64
    s, keys, _ = batch(82, dtype, seqs, h_kv * g, h_kv, 128, page, E4M3)
    see, qpos, kpos = sees(m, cached)
    for given in (True, False):  # (else the pages hold the call's own rows, from the call before)
        outs = []
        for fill in (0, 0x7F):
            x = {n: t.to(dev) for n, t in s.items()}
            if not given:
                paged_step(**x)
            for n in ("k_pages", "v_pages"):
                flat = x[n].view(I8)
                for b in range(4):
                    at = cached if given else cached + m
                    if at % page:
                        flat[int(s["table"][b, at // page]), at % page:] = fill
            if not given:
                x["k"] = x["v"] = None
            outs.append(paged_step(**x, max_new=m, max_len=cached + m, check=True))
        assert torch.equal(*outs), given
        for b in range(4):
            full = keys[b]
            if not given:
                full = [torch.cat([t[:cached], values(*held(t[cached:].to(dtype), E4M3))]) for t in full]
            check(outs[0][b * m:(b + 1) * m], *attend_set(s["q"][b * m:(b + 1) * m], *full, see, qpos, kpos)["out"], f"{given} {b}")


@pytest.mark.parametrize("hold", [I8, E4M3])
@pytest.mark.parametrize("d", [128, 64, 72])
@pytest.mark.parametrize("cap,bias", [(0.0, True), (3000.0, False), (3000.0, True), (5.0, False)])
def test_chunks_of_every_rule(dev, hold, d, cap, bias):
    """Chunks whose tiles are codes alone, some of the call's own rows or both, with one, two and four waves that
    share rows (528 blocks of 128 rows; 65 sequences; one)."""
    from tests.test_gpu_bounded_cache import test_step

    cases = [([(301, 700), (60, 33)], 8, 2, 0), ([(301, 200), (60, 0)], 8, 2, 97)]
    if d == 128:
        cases += [([(128, 3 * i % 40) for i in range(66)], 8, 2, 0), ([(40, 60 + i) for i in range(64)] + [(5, 60)], 16, 4, 0)]
    for seqs, h_q, h_kv, window in cases:
        test_step(dev, (BF16, hold, seqs, False, h_q, h_kv, d, 16, window, 5 if window else 0, cap, bias))


@pytest.mark.parametrize("hold", [I8, E4M3])
@pytest.mark.parametrize("m,trees", [(1, False), (2, False), (2, True)])
def test_one_and_two_tokens_around_borders_between_parts(dev, hold, m, trees):
    """The own rows of calls that few_codes takes, wherever the last part begins, and with codes for NaN in rows
    of the window's first page that nobody sees; and the same calls with their rows in the pages already."""
    from ssa_amd import paged_step
    from tests.cache_oracle import attend_set, held, sees, values
    from tests.dense_oracle import check
    from tests.test_gpu_bounded_cache import batch

    for window, g, d in ((0, 4, 128), (300, 8, 64), (520, 1, 128)):
        for cached in [*range(248, 264), *range(504, 520, 3), *range(1016, 1032, 5)]:
            s, keys, parents = batch(83, BF16, [(m, cached), (m, 3)], 2 * g, 2, d, 8, hold, window, 0, trees=trees)
            if window:
                lo = max(0, cached + 1 - window)
                for j in range(lo // 8 * 8, lo):
                    s["v_scales"][s["table"][0, j // 8], j % 8] = math.nan
            slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / (2 * g)) for i in range(2 * g)])
            kw = dict(window=window or None, slopes=slopes.to(dev), max_new=m, check=True)
            x = {n: t.to(dev) for n, t in s.items()}
            out = paged_step(**x, **kw)
            x["k"] = x["v"] = None
            again = paged_step(**x, **kw)
            for b, c in enumerate((cached, 3)):
                see, qpos, kpos = sees(m, c, parents[b], window, 0)
                rows = slice(b * m, (b + 1) * m)
                check(out[rows], *attend_set(s["q"][rows], *keys[b], see, qpos, kpos, 0.0, slopes)["out"], f"{window} {c}")
                full = [torch.cat([t[:c], values(*held(t[c:].to(BF16), hold))]) for t in keys[b]]
                check(again[rows], *attend_set(s["q"][rows], *full, see, qpos, kpos, 0.0, slopes)["out"], f"{window} {c} held")


@pytest.mark.parametrize("hold", [I8, E4M3])
@pytest.mark.parametrize("seqs,trees,h_q,h_kv,d,page,window,sinks,cap,bias", [
    ([(1, 31), (1, 32), (1, 33), (1, 500), (0, 40), (1, 127), (1, 0)], False, 8, 2, 128, 16, 0, 0, 0.0, False),
    ([(2, 1000), (1, 77), (2, 1), (2, 63)], False, 32, 4, 128, 64, 0, 0, 4.0, True),
    ([(1, 3000), (1, 100), (1, 2047)], False, 16, 1, 128, 128, 0, 0, 0.0, False),
    ([(2, 90), (1, 0), (2, 700)], False, 8, 2, 64, 8, 0, 0, 2000.0, True),
    ([(1, 500), (1, 70)], False, 2, 1, 8, 8, 0, 0, 0.0, True),
    ([(2, 100), (2, 1), (1, 33)], True, 4, 2, 24, 16, 0, 0, 0.0, True),
    ([(1, 600), (1, 0)], False, 16, 1, 112, 32, 0, 0, 3.0, False),
    ([(2, 300), (2, 1030), (2, 0)], True, 6, 2, 80, 16, 0, 0, 0.0, True),
    ([(2, 60), (2, 3), (1, 520)], True, 8, 8, 64, 8, 9, 5, 2000.0, True),
    ([(1, 5000), (1, 40), (1, 900)], False, 14, 1, 128, 32, 300, 40, 0.0, True),
    ([(2, 5000), (2, 40), (2, 900)], True, 8, 1, 128, 8, 1, 1, 0.0, False),
    ([(1, 900 + 37 * i) for i in range(40)], False, 8, 2, 64, 64, 0, 0, 5.0, False)])
def test_one_and_two_tokens_over_codes(dev, hold, seqs, trees, h_q, h_kv, d, page, window, sinks, cap, bias):
    """Calls that few_codes takes: outputs, the pages' new rows, and rows of no sequence."""
    from ssa_amd import paged_step
    from tests.dense_oracle import check
    from tests.test_gpu_bounded_cache import batch, bits, expect, pools_after

    s, keys, parents = batch(84, BF16, seqs, h_q, h_kv, d, page, hold, window, sinks, trees, behind=2)
    slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)]) if bias else None
    x = {n: t.to(dev) for n, t in s.items()}
    T = int(s["starts"][-1])
    out = paged_step(**x, softcap=cap or None, slopes=None if slopes is None else slopes.to(dev), window=window or None, sinks=sinks,
                     max_new=max(m for m, _ in seqs), max_len=max(m + c for m, c in seqs), check=True)
    assert not out[T:].any()
    for b, at, m, (value, bound) in expect(s, keys, parents, seqs, cap=cap, slopes=slopes, window=window, sinks=sinks):
        check(out[at:at + m], value, bound, f"sequence {b}")
    for name, want in pools_after(s, seqs, page, hold).items():
        assert torch.equal(bits(x[name].cpu()), bits(want)), name


@pytest.mark.parametrize("window,sinks", [(1 << 70, 0), (3, 1 << 70), (1 << 31, 1 << 31), (1, 1 << 63)])
def test_windows_and_first_keys_past_every_key(dev, window, sinks):
    """They see what a step without them does."""
    from ssa_amd import PagedKVCache, paged_step
    from tests.test_gpu_bounded_cache import batch

    for hold in (None, I8):
        s, _, _ = batch(85, BF16, [(3, 70), (1, 300), (60, 9)], 4, 2, 64, 16, hold)
        outs = []
        for kw in ({}, dict(window=window, sinks=sinks)):
            x = {n: t.to(dev) for n, t in s.items()}
            outs.append(paged_step(**x, check=True, **kw))
        assert torch.equal(*outs)
    x = [torch.randn(40, h, 64, device=dev, dtype=BF16, generator=torch.Generator(device=dev).manual_seed(1)) for h in (4, 2, 2)]
    outs = []
    for kw in ({}, dict(window=window, sinks=sinks)):
        cache = PagedKVCache(10, 16, 2, 64, **kw)
        a = cache.add()
        outs.append(torch.cat([cache.step(*x, [a], [40]), cache.step(*[t[:1] for t in x], [a], [1])]))
        assert cache.free_pages == 7
    assert torch.equal(*outs)
