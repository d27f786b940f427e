"""masked_attention of rows that see two key intervals, and mask_spans' windows, against the
64-bit oracle (tests/cache_oracle.py)."""

import math
import random

import pytest
import torch

from tests.cache_oracle import attend_set
from tests.dense_oracle import check

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def window_sees(n, n_q, pos0, window, sinks, starts=None, prefix=None):
    """[n_q, n]: row by row from the definition."""
    see = torch.zeros(n_q, n, dtype=torch.bool)
    for i in range(n_q):
        pos, a, e, pre = pos0 + i, 0, n, prefix[0] if prefix is not None and starts is None else 0
        if starts is not None:
            inside = [x for x in range(len(starts) - 1) if starts[x] <= pos < starts[x + 1]]
            if not inside:
                continue
            a, e = starts[inside[0]], min(starts[inside[0] + 1], n)
            pre = prefix[inside[0]] if prefix is not None else 0
        for lo, hi in ((max(a, pos - window + 1), min(pos + 1, e)), (a, min(a + sinks, pos + 1, e)), (a, min(a + pre, e))):
            see[i, max(lo, 0):max(hi, 0)] = True
    return see


def sets_see(spans, n):
    j = torch.arange(n)
    x = spans.long()
    return ((j >= x[:, :1]) & (j < x[:, 1:2])) | ((j >= x[:, 2:3]) & (j < x[:, 3:4]))


def run(dev, q, k, v, spans, see, pos0, cap=0.0, slopes=None, dout=None):
    """masked_attention and its gradients of a batch against the oracle."""
    from ssa_amd import masked_attention

    kw = dict(softcap=cap or None, slopes=None if slopes is None else slopes.to(dev), q_pos0=pos0)
    x = [t.to(dev).requires_grad_(dout is not None) for t in (q, k, v)]
    out = masked_attention(*x, spans, **kw)
    got = {"out": out.detach()}
    if dout is not None:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, dout.to(dev))))
    n, n_q = k.shape[1], q.shape[1]
    for b in range(len(q)):
        want = attend_set(q[b], k[b], v[b], see[b], pos0 + torch.arange(n_q), torch.arange(n), cap, slopes,
                          None if dout is None else dout[b])
        for name, (value, bound) in want.items():
            check(got[name][b], value, bound, f"{name} of sequence {b}")
    return got


CASES = [
    # dtype, B, n, n_q, h_q, h_kv, d, window, sinks, starts, prefix, cap, bias
    (F32, 1, 1, 1, 1, 1, 8, 1, 0, None, None, 0.0, False),
    (F32, 1, 203, 203, 8, 2, 64, 50, 4, None, None, 0.0, False),
    (BF16, 2, 130, 130, 4, 2, 64, 1, 1, None, None, 0.0, True),
    (BF16, 1, 700, 700, 8, 2, 128, 64, 16, None, None, 0.0, False),
    (BF16, 2, 333, 333, 6, 2, 96, 33, 100, [[0, 90, 91, 300], [5, 40, 333, 333]], None, 4.0, True),
    (F32, 2, 257, 257, 4, 4, 128, 31, 5, [[0, 100, 257], [20, 140, 200]], [[30, 0], [12, 70]], 2.0, True),
    (F32, 1, 400, 100, 8, 2, 64, 77, 40, None, None, 0.0, False),
    (BF16, 1, 1100, 60, 16, 2, 64, 200, 3, [[0, 1000, 1100]], None, 0.0, False),
    (BF16, 1, 1500, 1500, 4, 1, 128, 200, 130, None, [[300]], 0.0, False),
    (BF16, 1, 2100, 2100, 2, 2, 64, 100, 4, None, None, 0.0, False),
    (BF16, 3, 90, 90, 28, 4, 128, 1000, 7, None, None, 5.0, False),
    (F32, 1, 1300, 1300, 2, 1, 64, 128, 64, None, None, 0.0, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_windows(dev, case):
    from ssa_amd import mask_spans

    dtype, B, n, n_q, h_q, h_kv, d, window, sinks, starts, prefix, cap, bias = case
    print(f"window {case}", flush=True)
    g = torch.Generator().manual_seed(71)
    q, k, v = (torch.randn(B, m, h, d, generator=g).to(dtype) for m, h in ((n_q, h_q), (n, h_kv), (n, h_kv)))
    dout = torch.randn(B, n_q, h_q, d, generator=g).to(dtype)
    slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)]) if bias else None
    pos0 = n - n_q
    t = lambda x: None if x is None else torch.tensor(x, device=dev)  # noqa: E731
    spans = mask_spans(n, B, doc_starts=t(starts), prefix_lens=t(prefix), window=window, sinks=sinks, num_queries=n_q, device=dev)
    see = torch.stack([window_sees(n, n_q, pos0, window, sinks, starts and starts[b], prefix and prefix[b]) for b in range(B)])
    assert spans.shape == (B, n_q, 4)
    for b in range(B):
        x = spans[b].cpu()
        assert torch.equal(sets_see(x, n), see[b])
        one, two = x[:, 1] > x[:, 0], x[:, 3] > x[:, 2]
        assert (one | ~two).all() and (x[two, 3] < x[two, 0]).all(), "ascending, apart"
    run(dev, q, k, v, spans, see, pos0, cap, slopes, dout)


@pytest.mark.parametrize("dtype,d,n,h_q,h_kv,cap", [(F32, 64, 300, 4, 2, 0.0), (F32, 128, 200, 2, 2, 3.0), (BF16, 64, 600, 4, 1, 0.0),
                                                    (BF16, 128, 500, 8, 2, 0.0), (BF16, 72, 260, 2, 1, 2.0)])
def test_any_two_intervals(dev, dtype, d, n, h_q, h_kv, cap):
    """Pairs in any order, overlapping, empty, past the ends; rows that see nothing."""
    g, r = torch.Generator().manual_seed(72), random.Random(72)
    spans = torch.zeros(2, n, 4, dtype=torch.int32)
    for b in range(2):
        for i in range(n):
            pairs = []
            for _ in range(2):
                a = r.randrange(-20, n)
                pairs += [a, a + r.choice([-5, 0, 1, 3, 40, 64, n])]
            spans[b, i] = torch.tensor(pairs)
    spans[0, 10:50], spans[1, :70] = 0, torch.tensor([5, 5, n, n + 9], dtype=torch.int32)
    spans[0, 60] = torch.tensor([-(1 << 31), (1 << 31) - 1, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32)
    see = torch.stack([sets_see(x, n) for x in spans])
    q, k, v, dout = (torch.randn(2, n, h, d, generator=g).to(dtype) for h in (h_q, h_kv, h_kv, h_q))
    got = run(dev, q, k, v, spans.to(dev), see, 0, cap, None, dout)
    assert not got["out"][0, 10:50].any() and not got["dq"][1, :70].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,h_q,h_kv,d,window,sinks", [(3000, 8, 8, 64, 60, 3), (2600, 4, 1, 128, 100, 200), (5000, 2, 1, 64, 30, 1)])
def test_first_keys_of_long_sequences(dev, dtype, n, h_q, h_kv, d, window, sinks):
    """The first keys are seen by every row: their gradients come in parts."""
    from ssa_amd import mask_spans

    g = torch.Generator().manual_seed(73)
    q, k, v, dout = (torch.randn(1, n, h, d, generator=g).to(dtype) for h in (h_q, h_kv, h_kv, h_q))
    spans = mask_spans(n, window=window, sinks=sinks, device=dev)
    see = window_sees(n, n, 0, window, sinks)[None]
    run(dev, q, k, v, spans, see, 0, dout=dout)


def test_against_differences(dev):
    """Gradients against differences of the forward in 64 bits (the oracle's own)."""
    g = torch.Generator().manual_seed(74)
    n, d = 40, 8
    q, k, v, dout = (torch.randn(n, h, d, generator=g) for h in (2, 1, 1, 2))
    see = window_sees(n, n, 0, 7, 3)
    pos = torch.arange(n)
    slopes = torch.tensor([0.5, 0.1])
    want = attend_set(q, k, v, see, pos, pos, 2.0, slopes, dout)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        step = torch.randn(t.shape, generator=g).double() * 1e-6
        side = []
        for sign in (1.0, -1.0):
            x = {"dq": q.double(), "dk": k.double(), "dv": v.double()}
            x[name] = x[name] + sign * step
            side.append((attend_set(x["dq"], x["dk"], x["dv"], see, pos, pos, 2.0, slopes, r=0.0)["out"][0] * dout.double()).sum())
        slope = float((side[0] - side[1]) / 2)
        assert abs(slope - float((want[name][0] * step).sum())) <= 1e-5 * float(step.norm())
    from ssa_amd import mask_spans

    run(dev, q[None], k[None], v[None], mask_spans(n, window=7, sinks=3, device=dev), see[None], 0, 2.0, slopes, dout[None])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_hidden_and_visible_values_that_are_not_finite(dev, dtype):
    from ssa_amd import mask_spans, masked_attention

    n, window, sinks = 500, 40, 3
    g = torch.Generator().manual_seed(75)
    q, k, v, dout = (torch.randn(1, n, h, 64, generator=g).to(dtype) for h in (4, 2, 2, 4))
    spans = mask_spans(n, window=window, sinks=sinks, device=dev)
    see = window_sees(n, n, 0, window, sinks)
    pos = torch.arange(n)
    for j in (1, 7, 300):
        kk, vv = k.clone(), v.clone()
        kk[0, j], vv[0, j] = math.nan, math.inf
        x = [t.to(dev).requires_grad_(True) for t in (q, kk, vv)]
        out = masked_attention(*x, spans)
        free = ~see[:, j]
        dz = dout.clone()
        dz[0, ~free] = 0
        grads = torch.autograd.grad(out, x, dz.to(dev))
        want = attend_set(q[0][free], k[0], v[0], see[free], pos[free], pos, dout=dout[0][free])
        assert torch.isnan(out[0].cpu()[~free]).all()
        if free.any():
            check(out[0].detach()[free.to(dev)], *want["out"], "rows that do not see it")
            check(grads[0][0][free.to(dev)], *want["dq"], "their dq")
        # a key that only rows without it see has their gradients alone
        alone = [int(x) for x in ((see & ~free[:, None]).sum(0) == 0).nonzero()[:, 0] if see[:, x].any()]
        if alone:
            for i, name in ((1, "dk"), (2, "dv")):
                check(grads[i][0][alone], want[name][0][alone], want[name][1][alone], name)


def test_same_bits_streams_and_graphs(dev):
    from ssa_amd import mask_spans, masked_attention

    n = 1500
    g = torch.Generator().manual_seed(76)
    x = [torch.randn(1, n, h, 64, generator=g).to(BF16).to(dev).requires_grad_(True) for h in (8, 2, 2)]
    dout = torch.randn(1, n, 8, 64, generator=g).to(BF16).to(dev)

    def step():
        spans = mask_spans(n, window=64, sinks=5, device=dev)
        out = masked_attention(*x, spans)
        return (out.detach(), *torch.autograd.grad(out, x, dout))

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
    for _ in range(3):
        with torch.no_grad():
            x[0].add_(0.1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, step()))


def test_layouts_and_rejects(dev):
    from ssa_amd import mask_spans, masked_attention

    n, g = 150, torch.Generator().manual_seed(77)
    q, k, v, dout = (torch.randn(1, h, n, 64, generator=g).transpose(1, 2) for h in (4, 2, 2, 4))
    spans = mask_spans(n, window=20, sinks=2, device=dev)
    see = window_sees(n, n, 0, 20, 2)[None]
    run(dev, q, k, v, spans, see, 0, dout=dout)
    # unbatched, and float16 (widened)
    out = masked_attention(q[0].half().to(dev), k[0].half().to(dev), v[0].half().to(dev), spans[0])
    value, bound = attend_set(q[0].half(), k[0].half(), v[0].half(), see[0], torch.arange(n), torch.arange(n), r=0.0)["out"]
    check(out, value, bound + 2.0 ** -11 * (value.abs() + bound) + 2.0 ** -25, "fp16")
    x = [t.to(dev) for t in (q, k, v)]
    with pytest.raises(ValueError, match="spans"):
        masked_attention(*x, spans[:, :, :3].contiguous())
    with pytest.raises(ValueError, match="16 bytes"):
        masked_attention(*x, torch.zeros(4 * n + 2, device=dev, dtype=torch.int32)[2:].view(1, n, 4))
    with pytest.raises(ValueError, match="window"):
        mask_spans(n, window=0, device=dev)
    with pytest.raises(ValueError, match="causal"):
        mask_spans(n, window=4, causal=False, device=dev)
    with pytest.raises(ValueError, match="sinks"):
        mask_spans(n, sinks=2, device=dev)
    with pytest.raises(ValueError, match="sinks"):
        mask_spans(n, window=4, sinks=-1, device=dev)
    # no rows, no keys
    assert masked_attention(x[0][:, :0], x[1], x[2], spans[:, :0]).shape == (1, 0, 4, 64)
    none = masked_attention(x[0], x[1][:, :0], x[2][:, :0], spans, q_pos0=0)
    assert none.shape == q.shape and not none.any()


def test_windows_past_every_key(dev):
    """A window and first keys past 32 bits see what causal rows do."""
    from ssa_amd import mask_spans, masked_attention

    n, g = 200, torch.Generator().manual_seed(78)
    x = [torch.randn(1, n, h, 64, generator=g).to(dev) for h in (4, 2, 2)]
    want = masked_attention(*x)
    for window, sinks in ((1 << 40, 0), (n, 0), (1, 1 << 40), (7, n), ((1 << 31) - 1, (1 << 31) - 1)):
        assert torch.equal(masked_attention(*x, mask_spans(n, window=window, sinks=sinks, device=dev)), want)
