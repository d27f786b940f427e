"""paged_step and PagedKVCache against the 64-bit oracle (tests/dense_oracle.py)."""

import math

import pytest
import torch

from tests.dense_oracle import attend, check, spans_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _batch(seed, dtype, seqs, h_q, h_kv, d, page, spare=2, behind=0):
    """Sequences (new, cached) with scattered pages; rows and keys of nobody hold NaN."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-(m + c) // page) for m, c in seqs]
    pages = sum(counts) + spare
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), max(max(counts), 1) + 1), 10 ** 6, dtype=torch.int32)
    kp = torch.full((pages, page, h_kv, d), math.nan, dtype=dtype)
    vp = kp.clone()
    keys, at = [], 0
    for b, (m, c) in enumerate(seqs):
        mine = perm[at:at + counts[b]]
        at += counts[b]
        table[b, :counts[b]] = mine.to(torch.int32)
        k, v = (torch.randn(c + m, h_kv, d, generator=g).to(dtype) for _ in range(2))
        j = torch.arange(c)
        kp[mine[j // page], j % page], vp[mine[j // page], j % page] = k[:c], v[:c]
        keys.append((k, v))
    T = sum(m for m, _ in seqs)
    q = torch.randn(T + behind, h_q, d, generator=g).to(dtype)
    new = [torch.cat([x[i][c:] for x, (_, c) in zip(keys, seqs)] + [torch.full((behind, h_kv, d), math.nan, dtype=dtype)])
           for i in range(2)]
    starts = torch.tensor([sum(m for m, _ in seqs[:i]) for i in range(len(seqs) + 1)], dtype=torch.int32)
    return dict(q=q, k=new[0], v=new[1], k_pages=kp, v_pages=vp, table=table, starts=starts,
                cached=torch.tensor([c for _, c in seqs], dtype=torch.int32)), keys


def _expect(s, keys, seqs, cap, slopes):
    at = 0
    for b, (m, c) in enumerate(seqs):
        if m:
            yield b, at, m, attend(s["q"][at:at + m], *keys[b], spans_of(c + m, m, c), cap, slopes, c)["out"]
        at += m


CASES = [
    # dtype, sequences (new, cached), h_q, h_kv, d, page, cap, bias
    (F32, [(1, 0)], 2, 1, 8, 8, 0.0, False),
    (BF16, [(1, 0)], 1, 1, 64, 16, 0.0, True),
    (F32, [(1, 203)], 8, 2, 64, 16, 0.0, False),
    (BF16, [(1, 31), (1, 32), (1, 33), (1, 500), (0, 40), (1, 127)], 8, 2, 128, 16, 0.0, False),
    (BF16, [(1, 1000), (3, 77), (2, 1)], 28, 4, 128, 64, 4.0, True),
    (F32, [(2, 300), (1, 5)], 16, 1, 128, 32, 3.0, True),
    (BF16, [(5, 90), (6, 0), (8, 700)], 8, 2, 80, 8, 0.0, False),
    (BF16, [(1, 3000)], 16, 2, 64, 128, 0.0, True),
    (BF16, [(70, 200)], 8, 2, 64, 16, 0.0, False),
    (BF16, [(150, 0)], 4, 4, 128, 32, 0.0, False),
    (F32, [(40, 100), (1, 64), (33, 0)], 6, 2, 96, 16, 2.0, False),
    (BF16, [(1, 600), (45, 2000), (0, 0), (1, 9), (130, 31)], 28, 4, 128, 32, 5.0, True),
    (BF16, [(33, 1500)], 1, 1, 128, 64, 0.0, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_step(dev, case):
    from ssa_amd import paged_step

    dtype, seqs, h_q, h_kv, d, page, cap, bias = case
    slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)]) if bias else None
    s, keys = _batch(31, dtype, seqs, h_q, h_kv, d, page, behind=3)
    print(f"paged {case}", flush=True)
    x = {n: t.to(dev) for n, t in s.items()}
    out = torch.full(x["q"].shape, 7.0, device=dev, dtype=dtype)
    kw = dict(softcap=cap or None, slopes=None if slopes is None else slopes.to(dev), check=True)
    got = paged_step(**x, out=out, **kw)
    assert got is out
    T = int(s["starts"][-1])
    assert (out[T:] == 7).all(), "rows behind the last sequence"
    for b, at, m, (value, bound) in _expect(s, keys, seqs, cap, slopes):
        check(out[at:at + m], value, bound, f"sequence {b}")
    # the pools hold the new rows, and nothing else of them changed
    kp, vp = s["k_pages"].clone(), s["v_pages"].clone()
    for b, (m, c) in enumerate(seqs):
        j = torch.arange(c, c + m)
        pg = s["table"][b].long()[j // page]
        kp[pg, j % page], vp[pg, j % page] = keys[b][0][c:], keys[b][1][c:]
    for a, b in ((x["k_pages"], kp), (x["v_pages"], vp)):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    # the keys are there now: the same without k and v, and with tight bounds
    x["k"] = x["v"] = None
    again = paged_step(**x, max_new=max(max(m for m, _ in seqs), 1), max_len=max(m + c for m, c in seqs), **kw)
    for b, at, m, (value, bound) in _expect(s, keys, seqs, cap, slopes):
        check(again[at:at + m], value, bound, f"sequence {b} without append")


def test_strided_pools_and_rows(dev):
    """Pools as [pages, h_kv, page, d] and q, k, v cut out of one projection."""
    from ssa_amd import paged_step

    seqs, h_q, h_kv, d, page = [(1, 50), (20, 40)], 4, 2, 64, 16
    s, keys = _batch(32, BF16, seqs, h_q, h_kv, d, page)
    x = {n: t.to(dev) for n, t in s.items()}
    want = paged_step(**{**x, "k_pages": x["k_pages"].clone(), "v_pages": x["v_pages"].clone()})
    for n in ("k_pages", "v_pages"):
        x[n] = x[n].transpose(1, 2).contiguous().transpose(1, 2)
    qkv = torch.cat((x["q"], x["k"], x["v"]), 1)
    x["q"], x["k"], x["v"] = qkv[:, :h_q], qkv[:, h_q:h_q + h_kv], qkv[:, h_q + h_kv:]
    wide = torch.zeros(x["table"].shape[0], x["table"].shape[1] + 5, device=dev, dtype=torch.int32)
    wide[:, :x["table"].shape[1]] = x["table"]
    x["table"] = wide[:, :x["table"].shape[1]]
    assert torch.equal(paged_step(**x), want)


@pytest.mark.parametrize("dtype,h_q,h_kv,d", [(F32, 4, 2, 64), (F32, 4, 2, 128), (BF16, 8, 2, 64), (BF16, 6, 2, 96)], ids=str)
@pytest.mark.parametrize("cap,bias", [(0.0, False), (3.0, False), (3.0, True)])
def test_prompts(dev, dtype, h_q, h_kv, d, cap, bias):
    """Prompts, most of whose keys are the call's own rows: cut out of one projection, behind
    nothing, behind an odd number of cached keys and behind whole tiles; rows behind the last."""
    from ssa_amd import paged_step

    seqs, page = [(300, 0), (131, 37), (65, 128), (1, 0)], 16
    s, keys = _batch(42, dtype, seqs, h_q, h_kv, d, page, behind=2)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(h_q)]) if bias else None
    x = {n: t.to(dev) for n, t in s.items()}
    qkv = torch.cat((x["q"], x["k"], x["v"]), 1)
    x["q"], x["k"], x["v"] = qkv[:, :h_q], qkv[:, h_q:h_q + h_kv], qkv[:, h_q + h_kv:]
    out = paged_step(**x, softcap=cap or None, slopes=slopes.to(dev) if bias else None, max_new=300, max_len=300, check=True)
    for b, at, m, (value, bound) in _expect(s, keys, seqs, cap, slopes):
        check(out[at:at + m], value, bound, f"sequence {b}")
    for b, (m, c) in enumerate(seqs):  # and they are in their pages
        j = torch.arange(c + m)
        for pool, want in zip((x["k_pages"], x["v_pages"]), keys[b]):
            got = pool.cpu()[s["table"][b].long()[j // page], j % page]
            assert torch.equal(got, want)


def test_values_in_unwritten_rows(dev):
    """_batch leaves NaN in rows of the pages that hold no key: the outputs are finite (test_step);
    a NaN that a sequence does hold reaches its tokens and no other sequence's."""
    from ssa_amd import paged_step

    seqs = [(1, 100), (1, 100), (40, 100)]
    for dtype in (F32, BF16):
        s, _ = _batch(33, dtype, seqs, 4, 2, 64, 16)
        s["v_pages"][s["table"][1, 2], 3, 0, 9] = math.nan
        out = paged_step(**{n: t.to(dev) for n, t in s.items()}).cpu()
        bad = torch.isnan(out)
        assert bad[1, :2, 9].all() and bad.sum() == 2


def test_bad_sequences_are_left_out(dev):
    from ssa_amd import paged_step

    seqs, page = [(1, 40), (2, 30), (1, 20)], 16
    s, keys = _batch(34, BF16, seqs, 4, 2, 64, page)
    for breakage in ("cached", "negative", "bound", "page"):
        x = {n: t.clone().to(dev) for n, t in s.items()}
        kw = {}
        if breakage == "cached":
            x["cached"][1] = 10 ** 6
        elif breakage == "negative":
            x["cached"][1] = -1
        elif breakage == "bound":
            kw["max_new"] = 1
        else:
            x["table"][1, 0] = 10 ** 8
        out = torch.full(x["q"].shape, 7.0, device=dev, dtype=BF16)
        with pytest.raises(IndexError):
            paged_step(**x, out=out, check=True, **kw)
        if breakage != "page":
            assert (out[1:3] == 7).all()
        for b, at, m, (value, bound) in _expect(s, keys, seqs, 0.0, None):
            if b != 1:
                check(out[at:at + m], value, bound, f"{breakage}: sequence {b}")


def test_captured_and_on_streams(dev):
    """A captured step follows lengths, tables and tokens; the split call, twice at once."""
    from ssa_amd import paged_step

    seqs = [(1, 900), (1, 250), (1, 64)]
    s, _ = _batch(35, BF16, seqs, 8, 2, 128, 16)
    x = {n: t.to(dev) for n, t in s.items()}
    kw = dict(max_new=1, max_len=1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_step(**x, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_step(**x, **kw)
    with torch.cuda.graph(other):
        out2 = paged_step(**x, **kw)
    for step in range(4):
        with torch.no_grad():
            x["q"].add_(0.25)
            x["k"].mul_(0.9)
            if step:
                x["cached"].sub_(7)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        eager = paged_step(**x, **kw)
        assert torch.equal(out, eager) and torch.equal(out2, eager)
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = paged_step(**{**x, "k": None, "v": None}, **kw)
    torch.cuda.synchronize()
    got = []
    for st in streams * 3:
        with torch.cuda.stream(st):
            got.append(paged_step(**{**x, "k": None, "v": None}, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_far_pages(dev):
    """Pages past 2^31 elements and 2^32 bytes of the pool."""
    from ssa_amd import paged_step

    page, h_kv, d = 64, 8, 128
    pages = (1 << 32) // (page * h_kv * d * 2) + 40
    k_pages = torch.zeros(pages, page, h_kv, d, device=dev, dtype=BF16)
    v_pages = torch.zeros_like(k_pages)
    seqs = [(1, 300), (30, 100)]
    s, keys = _batch(36, BF16, seqs, 8, h_kv, d, page)
    small = s["k_pages"].shape[0]
    k_pages[pages - small:] = s["k_pages"].to(dev)
    v_pages[pages - small:] = s["v_pages"].to(dev)
    s["table"] = torch.where(s["table"] < small, s["table"] + pages - small, s["table"])
    x = {n: t.to(dev) for n, t in s.items()}
    x["k_pages"], x["v_pages"] = k_pages, v_pages
    out = paged_step(**x, check=True)
    for b, at, m, (value, bound) in _expect(s, keys, seqs, 0.0, None):
        check(out[at:at + m], value, bound, f"sequence {b}")


@pytest.mark.parametrize("m", [1, 40])
def test_shared_pages_and_rows_before_the_first_sequence(dev, m):
    """Sequences that share the pages of a prefix, one of which stands in it twice; rows before
    the first sequence and behind the last keep what they held."""
    from ssa_amd import paged_step

    page, h_q, h_kv, d = 16, 8, 2, 64
    s, keys = _batch(39, BF16, [(m, 64), (m, 64)], h_q, h_kv, d, page)
    pre = s["table"][0, :3]
    s["table"][0, 2] = pre[0]          # keys 32..47 are keys 0..15 again
    s["table"][1, :3] = s["table"][0, :3]
    for b in range(2):
        for x, pool in zip(keys[b], (s["k_pages"], s["v_pages"])):
            for i in range(3):
                x[16 * i:16 * i + 16] = pool[s["table"][0, i]]
    edge = 3
    for n in ("q", "k", "v"):
        nobody = torch.full((edge, *s[n].shape[1:]), math.nan, dtype=BF16)
        s[n] = torch.cat((nobody, s[n], nobody))
    s["starts"] += edge
    out = torch.full(s["q"].shape, 7.0, dtype=BF16, device=dev)
    paged_step(**{n: t.to(dev) for n, t in s.items()}, out=out, check=True)
    assert (out[:edge] == 7).all() and (out[-edge:] == 7).all()
    for b in range(2):
        rows = slice(edge + b * m, edge + (b + 1) * m)
        check(out[rows], *attend(s["q"][rows], *keys[b], spans_of(64 + m, m, 64), 0.0, None, 64)["out"], f"sequence {b}")


def test_bounds_past_the_tokens_and_the_table(dev):
    """max_new and max_len may say more than a sequence can hold."""
    from ssa_amd import paged_step

    s, _ = _batch(41, BF16, [(1, 300), (50, 70)], 8, 2, 64, 16)
    x = {n: t.to(dev) for n, t in s.items()}
    assert torch.equal(paged_step(**x, check=True), paged_step(**x, max_new=10 ** 6, max_len=10 ** 9, check=True))


def test_empty(dev):
    from ssa_amd import paged_step

    s, _ = _batch(37, F32, [(0, 20), (0, 0)], 2, 1, 16, 8)
    assert paged_step(**{n: t.to(dev) for n, t in s.items()}, check=True).shape == (0, 2, 16)


def test_rejects(dev):
    from ssa_amd import paged_step

    s, _ = _batch(38, F32, [(1, 20)], 2, 1, 16, 8)
    x = {n: t.to(dev) for n, t in s.items()}
    bad = [({"k": None}, ValueError, "together"), ({"table": x["table"].long()}, ValueError, "table"),
           ({"starts": x["starts"][:1]}, ValueError, "starts"), ({"cached": x["cached"].float()}, ValueError, "cached"),
           ({"q": x["q"].bfloat16()}, TypeError, "dtype"), ({"k": x["k"][:, :, :8]}, ValueError, "k must"),
           ({"k_pages": x["k_pages"][:, :7], "v_pages": x["v_pages"][:, :7]}, NotImplementedError, "page_size"),
           ({"softcap": -1.0}, ValueError, "softcap"), ({"max_new": 0}, RuntimeError, "max_new"),
           ({"starts": x["starts"].cpu()}, RuntimeError, "HIP"),
           ({"out": torch.empty(1, 2, 8, device=dev)}, ValueError, "out")]
    for change, err, text in bad:
        with pytest.raises(err, match=text):
            paged_step(**{**x, **change})


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_cache_and_the_operators_together(dev, dtype):
    """Rotated q and k of a prompt in one masked_attention call, and the same tokens served:
    chunks and single tokens of two sequences through PagedKVCache, other sequences coming and
    going in between.  Both within the oracle's bounds of the same values."""
    from ssa_amd import PagedKVCache, axis_rope_freqs, mask_spans, masked_attention, rope_axes

    h_q, h_kv, d, n = 8, 2, 64, 90
    g = torch.Generator().manual_seed(40)
    freqs = axis_rope_freqs(d, 1e4, dev)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(h_q)])
    data = []
    for i in range(2):
        q, k, v = (torch.randn(1, n, h, d, generator=g).to(dtype).to(dev) for h in (h_q, h_kv, h_kv))
        pos = torch.stack([torch.arange(n), torch.arange(n) // 7, torch.arange(n) % 7])[:, None].to(dev)
        q, k = rope_axes(q, k, pos, freqs, (8, 12, 12))
        data.append((q[0], k[0], v[0]))
    whole = [masked_attention(q, k, v, mask_spans(n, 1, device=dev)[0], softcap=6.0, slopes=slopes.to(dev)) for q, k, v in data]
    want = [attend(*(t.cpu() for t in x), spans_of(n, n, 0), 6.0, slopes)["out"] for x in data]
    for b in range(2):
        check(whole[b], *want[b], f"whole {b}")
    cache = PagedKVCache(16, 16, h_kv, d, dtype=dtype, device=dev)
    other = cache.add()
    junk = [torch.randn(40, h, d, generator=g).to(dtype).to(dev) for h in (h_q, h_kv, h_kv)]
    cache.step(*junk, [other], [40])
    seqs = [cache.add(), cache.add()]
    served = [[], []]
    at = [0, 0]
    for turn, counts in enumerate(((50, 1), (1, 33), (1, 1), (37, 54), (1, 1))):
        if turn == 2:
            cache.free(other)
        parts = [tuple(t[at[b]:at[b] + counts[b]] for t in data[b]) for b in range(2)]
        out = cache.step(*(torch.cat(t) for t in zip(*parts)), seqs, list(counts), softcap=6.0, slopes=slopes.to(dev))
        served[0].append(out[:counts[0]])
        served[1].append(out[counts[0]:])
        at = [at[b] + counts[b] for b in range(2)]
    assert [cache.length(s) for s in seqs] == [n, n] and cache.free_pages == 16 - 12
    for b in range(2):
        check(torch.cat(served[b]), *want[b], f"served {b}")
    with pytest.raises(ValueError, match="cache full"):
        cache.step(*(torch.cat([t] * 3) for t in data[0]), [seqs[0]], [3 * n])
    assert cache.free_pages == 4 and cache.length(seqs[0]) == n
    for s in seqs:
        cache.free(s)
    assert cache.free_pages == 16
    with pytest.raises(ValueError, match="not open"):
        cache.step(*data[0], [seqs[0]], [n])


@pytest.mark.parametrize("m", [1, 50])
def test_pools_with_whole_heads_apart(dev, m):
    """Pools as [h_kv, pages, page, d] and rows as [h, T, d]: heads more than 16 MiB apart."""
    from ssa_amd import paged_step

    h_q, h_kv, d, page = 4, 2, 64, 16
    s, keys = _batch(43, BF16, [(m, 100), (m, 30)], h_q, h_kv, d, page)
    x = {n: t.to(dev) for n, t in s.items()}
    want = paged_step(**{**x, "k_pages": x["k_pages"].clone(), "v_pages": x["v_pages"].clone()})
    step = (40 << 20) // 2
    for n in ("k_pages", "v_pages"):
        pool = torch.zeros(h_kv * step, device=dev, dtype=BF16)
        pages = torch.as_strided(pool, x[n].shape, (page * d, d, step, 1))
        x[n] = pages.copy_(x[n])
    for n in ("q", "k", "v"):
        rows = torch.zeros(h_q * step, device=dev, dtype=BF16)
        x[n] = torch.as_strided(rows, x[n].shape, (d, step, 1)).copy_(x[n])
    out = torch.as_strided(torch.zeros(h_q * step, device=dev, dtype=BF16), x["q"].shape, (d, step, 1))
    assert torch.equal(paged_step(**x, out=out, check=True), want)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 80)], ids=str)
@pytest.mark.parametrize("seqs", [[(1, 40), (1, 30), (90, 20), (70, 5), (3, 0)], [(1, 40), (1, 30), (2, 7), (3, 0)],
                                  [(1, 1500), (1, 30), (2, 7), (3, 0)], [(50, 2000), (40, 30), (1, 7), (3, 0)]], ids=str)
def test_rows_that_nothing_writes_are_zeros(dev, dtype, d, seqs):
    """Without ``out``: rows before the first sequence, behind the last and of sequences that are
    left out are zeros whatever the memory held; calls with and without chunks and parts."""
    from ssa_amd import paged_step

    h_q, h_kv, edge = 4, 2, 300
    s, keys = _batch(44, dtype, seqs, h_q, h_kv, d, 16, behind=edge)
    for n in ("q", "k", "v"):
        s[n] = torch.cat((torch.full((edge, *s[n].shape[1:]), math.nan, dtype=dtype), s[n]))
    s["starts"] += edge
    for b in (1, 2):
        s["cached"][b] = 10 ** 6
    x = {n: t.to(dev) for n, t in s.items()}
    stale = torch.full(x["q"].shape, 7.0, device=dev, dtype=dtype)  # the next tensor of this size takes its memory
    torch.cuda.synchronize()
    at = stale.data_ptr()
    del stale
    out = paged_step(**x)
    assert out.data_ptr() == at
    rows = torch.zeros(out.shape[0], dtype=torch.bool)
    for b, i, m, (value, bound) in _expect({**s, "q": s["q"][edge:]}, keys, seqs, 0.0, None):
        if b not in (1, 2):
            check(out[edge + i:edge + i + m], value, bound, f"sequence {b}")
            rows[edge + i:edge + i + m] = True
    assert (out.cpu()[~rows] == 0).all()
    none = {**x, "table": x["table"][:0], "starts": x["starts"][:1], "cached": x["cached"][:0]}
    assert (paged_step(**none) == 0).all()
    out.fill_(7.0)
    assert (paged_step(**none, out=out) == 7).all()


def test_expanded_tensors_are_not_written_to(dev):
    """Pools that hold one head for several take no new rows, but are read; out is a tensor of its own."""
    from ssa_amd import paged_step

    s, keys = _batch(45, BF16, [(1, 40), (2, 10)], 4, 2, 64, 16)
    x = {n: t.to(dev) for n, t in s.items()}
    paged_step(**x)
    one = {n: x[n][:, :, :1].expand(-1, -1, 2, -1) for n in ("k_pages", "v_pages")}
    with pytest.raises(ValueError, match="k_pages"):
        paged_step(**{**x, **one})
    with pytest.raises(ValueError, match="out"):
        paged_step(**x, out=torch.zeros(3, 1, 64, device=dev, dtype=BF16).expand(-1, 4, -1))
    got = paged_step(**{**x, **one, "k": None, "v": None})
    want = paged_step(**{**x, **{n: t.contiguous() for n, t in one.items()}, "k": None, "v": None})
    assert torch.equal(got, want)
