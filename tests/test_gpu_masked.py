"""masked_attention and mask_spans against the 64-bit oracle (tests/dense_oracle.py)."""

import math

import pytest
import torch

from tests.dense_oracle import attend, check, spans_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _inputs(seed, dtype, B, n_q, n, h_q, h_kv, d):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return make(B, n_q, h_q, d), make(B, n, h_kv, d), make(B, n, h_kv, d), make(B, n_q, h_q, d)


def _slopes(h_q):
    return torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)])


def _run(dev, q, k, v, dout, spans, cap=0.0, slopes=None, q_pos0=None, **kw):
    from ssa_amd import masked_attention

    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = masked_attention(*leaves, None if spans is None else spans.to(dev), softcap=cap or None,
                           slopes=None if slopes is None else slopes.to(dev), q_pos0=q_pos0, **kw)
    grads = torch.autograd.grad(out, leaves, dout.to(dev))
    with torch.no_grad():  # the call without gradients gives the same output
        again = masked_attention(*leaves, None if spans is None else spans.to(dev), softcap=cap or None,
                                 slopes=None if slopes is None else slopes.to(dev), q_pos0=q_pos0, **kw)
    assert torch.equal(out.detach().view(torch.uint8) if out.numel() else out, again.view(torch.uint8) if out.numel() else again)
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _check(res, q, k, v, dout, spans, cap, slopes, q_pos0, what=""):
    for b in range(q.shape[0]):
        want = attend(q[b], k[b], v[b], spans[b], cap, slopes, q_pos0, dout[b])
        for name, (value, bound) in want.items():
            check(res[name][b], value, bound, f"{what}{name}[{b}]")


CASES = [
    # dtype, B, n_q, n, h_q, h_kv, d, cap, bias
    (F32, 1, 1, 1, 1, 1, 8, 0.0, False),
    (BF16, 1, 1, 1, 2, 1, 8, 0.0, True),
    (F32, 2, 31, 31, 4, 2, 64, 0.0, False),
    (BF16, 2, 33, 33, 4, 2, 64, 0.0, False),
    (BF16, 1, 64, 64, 8, 2, 128, 0.0, False),
    (F32, 1, 65, 65, 6, 2, 96, 4.0, False),
    (BF16, 1, 127, 127, 7, 1, 128, 4.0, True),
    (BF16, 2, 129, 129, 4, 4, 80, 0.0, True),
    (F32, 1, 130, 130, 3, 1, 128, 0.0, True),
    (BF16, 1, 203, 203, 8, 2, 64, 2.0, False),
    (F32, 1, 203, 203, 8, 2, 64, 2.0, True),
    (BF16, 1, 257, 257, 16, 1, 64, 0.0, False),
    (BF16, 1, 40, 300, 4, 2, 128, 0.0, True),     # a block of queries behind cached keys
    (F32, 1, 17, 150, 4, 1, 72, 0.0, False),
    (BF16, 1, 2, 2100, 4, 2, 64, 0.0, True),      # few rows, many keys: split along the keys
    (F32, 1, 1, 1537, 2, 2, 128, 3.0, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("mask", ["causal", "full", "docs", "prefix"])
def test_forward_and_gradients(dev, case, mask):
    from ssa_amd import mask_spans

    dtype, B, n_q, n, h_q, h_kv, d, cap, bias = case
    q, k, v, dout = _inputs(17, *case[:7])
    slopes = _slopes(h_q) if bias else None
    p0 = n - n_q
    if mask == "causal":
        spans, dev_spans = [spans_of(n, n_q, p0)] * B, None
    elif mask == "full":
        spans = [spans_of(n, n_q, p0, causal=False)] * B
        dev_spans = mask_spans(n, B, causal=False, num_queries=n_q, device=dev)
    else:
        cuts = [[0, n // 5, n // 5, n // 2, n - n // 9], [n // 7, n // 3, n - 1, n, n]]
        starts = [cuts[b % 2] for b in range(B)]
        prefix = [[(s[i + 1] - s[i]) // 2 + i for i in range(4)] for s in starts] if mask == "prefix" else None
        spans = [spans_of(n, n_q, p0, True, starts[b], prefix[b] if prefix else None) for b in range(B)]
        dev_spans = mask_spans(n, B, doc_starts=torch.tensor(starts, device=dev, dtype=torch.int32), num_queries=n_q,
                               prefix_lens=None if prefix is None else torch.tensor(prefix, device=dev))
    if dev_spans is not None:
        assert torch.equal(dev_spans.cpu(), torch.stack(spans)), "mask_spans"
    print(f"masked {mask} {case}", flush=True)
    res = _run(dev, q, k, v, dout, dev_spans, cap, slopes)
    _check(res, q, k, v, dout, spans, cap, slopes, p0)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64), (BF16, 128)], ids=str)
def test_any_intervals(dev, dtype, d):
    """Intervals in no order, empty rows among them, and bounds past the keys."""
    B, n, h_q, h_kv = 2, 230, 4, 2
    q, k, v, dout = _inputs(3, dtype, B, n, n, h_q, h_kv, d)
    g = torch.Generator().manual_seed(4)
    lo = torch.randint(-40, n, (B, n, 1), generator=g)
    spans = torch.cat((lo, lo + torch.randint(-30, n, (B, n, 1), generator=g)), -1).to(torch.int32)
    want = spans.clamp(0, n)
    want = torch.where(want[..., 1:] > want[..., :1], want, 0)
    res = _run(dev, q, k, v, dout, spans)
    _check(res, q, k, v, dout, want, 0.0, None, 0)
    empty = (want[..., 0] == want[..., 1])
    assert empty.any() and (res["out"].cpu()[empty] == 0).all() and (res["dq"].cpu()[empty] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_nothing_visible(dev, dtype):
    q, k, v, dout = _inputs(5, dtype, 1, 70, 70, 4, 2, 64)
    res = _run(dev, q, k, v, dout, torch.zeros(1, 70, 2, dtype=torch.int32))
    for x in res.values():
        assert (x == 0).all()


@pytest.mark.parametrize("dtype,n,n_q", [(F32, 150, 150), (BF16, 150, 150), (BF16, 1600, 3)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_have_no_influence(dev, dtype, n, n_q, bad):
    """Rows and keys of the padding behind the documents hold anything; so do later tokens."""
    h_q, h_kv, d = 4, 2, 64
    q, k, v, dout = _inputs(6, dtype, 1, n_q, n, h_q, h_kv, d)
    p0 = n - n_q
    spans = spans_of(n, n_q, p0, starts=[0, n // 3, n - n_q // 3 - 20])
    hidden = torch.ones(n, dtype=torch.bool)
    for lo, hi in spans.tolist():
        hidden[lo:hi] = False
    dead = spans[:, 0] == spans[:, 1]
    assert hidden.any()
    k[0, hidden], v[0, hidden] = bad, bad
    q[0, dead], dout[0, dead] = bad, bad
    res = _run(dev, q, k, v, dout, spans[None])
    _check(res, q, k, v, dout, spans[None], 0.0, None, p0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_visible_values_that_are_not_finite(dev, dtype, bad):
    """A value that is not finite reaches the rows that see its key, and no others."""
    n = 100
    q, k, v, dout = _inputs(7, dtype, 1, n, n, 4, 2, 64)
    v[0, 60, 1, 5] = bad
    res = _run(dev, q, k, v, dout, None)
    out = res["out"].detach().cpu()[0]
    assert torch.isfinite(out[:60]).all() and torch.isfinite(out[:, :2]).all()
    assert not torch.isfinite(out[60:, 2:, 5]).any()
    assert torch.isfinite(out[60:, 2:, 6]).all()


def test_scores_of_minus_infinity(dev):
    """Keys that score -inf weigh nothing; a row whose every key does is NaN, as softmax makes it."""
    for dtype in (F32, BF16):
        q, k, v, dout = _inputs(8, dtype, 1, 40, 40, 2, 1, 64)
        q = q.abs() + 0.1
        k[0, 7] = -math.inf
        res = _run(dev, q, k, v, dout, None)
        out = res["out"].detach().cpu()
        assert torch.isfinite(out).all()
        kept = k.clone()
        kept[0, 7] = 0
        spans = spans_of(40, 40, 0)
        want = attend(q[0, :7], kept[0], v[0], spans[:7])["out"]
        check(out[0, :7], *want, "rows before the key")
        spans[:, 0], spans[:, 1] = 7, 8
        assert torch.isnan(_run(dev, q, k, v, dout, spans[None])["out"]).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_large_scores(dev, dtype):
    """Scores far past exp's range, and equal ones."""
    q, k, v, dout = _inputs(9, dtype, 1, 90, 90, 2, 2, 64)
    q = q * 64
    spans = spans_of(90, 90, 0)
    res = _run(dev, q, k, v, dout, None)
    _check(res, q, k, v, dout, spans[None], 0.0, None, 0)
    res = _run(dev, q * 0, k, v, dout, None)
    _check(res, q * 0, k, v, dout, spans[None], 0.0, None, 0)
    res = _run(dev, q, k, v, dout, None, cap=5.0)  # the cap saturates
    _check(res, q, k, v, dout, spans[None], 5.0, None, 0)


def test_layouts(dev):
    """Transposed and strided views, a broadcast head, rows off alignment, no batch, a scale."""
    from ssa_amd import masked_attention

    q, k, v, dout = _inputs(10, BF16, 2, 77, 77, 4, 2, 64)
    ref = _run(dev, q, k, v, dout, None)
    to_heads = lambda t: t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)  # noqa: E731
    wide = lambda t: torch.cat((t, t), -1).to(dev)[..., :64]  # noqa: E731
    odd = lambda t: torch.nn.functional.pad(t, (3, 2)).to(dev)[..., 3:67]  # noqa: E731
    for make in (to_heads, wide, odd):
        leaves = [make(t).detach().requires_grad_(True) for t in (q, k, v)]
        out = masked_attention(*leaves)
        grads = torch.autograd.grad(out, leaves, make(dout))
        for x, y in zip((out, *grads), ref.values()):
            assert torch.equal(x, y)
    one = masked_attention(q[1].to(dev), k[1].to(dev), v[1].to(dev))
    assert torch.equal(one, ref["out"][1])
    # a head of k and v broadcast over all: its gradient is the sum over its copies
    kb, vb = (t[:, :, :1].to(dev).detach().requires_grad_(True) for t in (k, v))
    out = masked_attention(q.to(dev), kb.expand(-1, -1, 4, -1), vb.expand(-1, -1, 4, -1))
    dk, dv = torch.autograd.grad(out, (kb, vb), dout.to(dev))
    for b in range(2):
        want = attend(q[b], k[b, :, :1], v[b, :, :1], spans_of(77, 77, 0), dout=dout[b])
        # (four partial gradients, each rounded once, are added in bf16: two more roundings)
        for got, name in ((dk, "dk"), (dv, "dv")):
            val, bound = want[name]
            parts = attend(q[b], k[b, :, :1].expand(-1, 4, -1), v[b, :, :1].expand(-1, 4, -1), spans_of(77, 77, 0),
                           dout=dout[b])[name]
            check(got[b], val, bound + 4 * 2.0 ** -8 * parts[0].abs().sum(1, keepdim=True) + parts[1].sum(1, keepdim=True), name)
    half = masked_attention(q[:1].half().to(dev), k[:1].half().to(dev), v[:1].half().to(dev), scale=3.0)
    assert half.dtype == torch.float16
    val, bound = attend(q[0].half(), k[0].half(), v[0].half(), spans_of(77, 77, 0), scale=3.0, round_to=F32)["out"]
    check(half[0], val, bound + 2.0 ** -11 * val.abs() + 2.0 ** -24, "fp16")


def test_same_bits_and_streams(dev):
    """No atomics: repeated calls, another stream and graph replays give the same bits."""
    from ssa_amd import mask_spans, masked_attention

    q, k, v, dout = (t.to(dev) for t in _inputs(11, BF16, 1, 300, 300, 8, 2, 64))
    starts = torch.tensor([[0, 120, 290]], device=dev, dtype=torch.int32)

    def step(q, k, v):
        spans = mask_spans(300, 1, doc_starts=starts)
        out = masked_attention(q, k, v, spans, softcap=20.0)
        return (out, *torch.autograd.grad(out, (q, k, v), dout))

    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    first = [t.detach().clone() for t in step(*leaves)]
    for a, b in zip(first, step(*leaves)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    # captured with leaves of its own
    mine = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*mine)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*mine)
    for shift in (0.0, 0.5, 0.0):
        with torch.no_grad():
            for m, t in zip(mine, (q, k, v)):
                m.copy_(t + shift)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(*[(t.detach() + shift).requires_grad_(True) for t in (q, k, v)])
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_two_graphs_and_two_calls_at_once(dev):
    """Split calls on two streams at once, each with a workspace of its own."""
    from ssa_amd import masked_attention

    sets = [[t.to(dev) for t in _inputs(20 + i, BF16, 1, 2, 4000, 8, 2, 128)[:3]] for i in range(2)]
    want = [masked_attention(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = masked_attention(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_empty_sizes(dev):
    from ssa_amd import mask_spans, masked_attention

    q, k, v, dout = _inputs(12, F32, 1, 0, 5, 2, 1, 16)
    res = _run(dev, q, k, v, dout, None)
    assert res["out"].shape == (1, 0, 2, 16) and (res["dk"] == 0).all() and (res["dv"] == 0).all()
    q, k, v, dout = _inputs(12, F32, 1, 5, 0, 2, 1, 16)
    res = _run(dev, q, k, v, dout, None, q_pos0=0)
    assert (res["out"] == 0).all() and (res["dq"] == 0).all()
    q, k, v, dout = _inputs(12, F32, 0, 5, 5, 2, 1, 16)
    assert masked_attention(q.to(dev), k.to(dev), v.to(dev)).shape == (0, 5, 2, 16)
    assert mask_spans(5, 0, device=dev).shape == (0, 5, 2)


def test_rejects(dev):
    from ssa_amd import mask_spans, masked_attention

    q, k, v, _ = (t.to(dev) for t in _inputs(13, F32, 1, 8, 8, 4, 2, 16))
    spans = mask_spans(8, 1, device=dev)
    with pytest.raises(ValueError, match="spans"):
        masked_attention(q, k, v, spans.long())
    with pytest.raises(ValueError, match="spans"):
        masked_attention(q, k, v, spans[:, :7])
    with pytest.raises(TypeError, match="dtype"):
        masked_attention(q, k.bfloat16(), v)
    with pytest.raises(ValueError, match="divisible"):
        masked_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError, match="k and v"):
        masked_attention(q, k, v[:, :5])
    with pytest.raises(ValueError, match="softcap"):
        masked_attention(q, k, v, softcap=0.0)
    with pytest.raises(RuntimeError, match="scale"):
        masked_attention(q, k, v, scale=0.0)
    with pytest.raises(ValueError, match="slopes"):
        masked_attention(q, k, v, slopes=torch.ones(3, device=dev))
    with pytest.raises(NotImplementedError, match="slopes"):
        masked_attention(q, k, v, slopes=torch.ones(4, device=dev, requires_grad=True))
    with pytest.raises(NotImplementedError, match="head_dim"):
        masked_attention(q[..., :12], k[..., :12], v[..., :12])
    with pytest.raises(RuntimeError, match="HIP"):
        masked_attention(q.cpu(), k.cpu(), v.cpu())
    with pytest.raises(RuntimeError, match="HIP"):
        masked_attention(q, k, v, spans.cpu())
    with pytest.raises(ValueError, match="prefix_lens"):
        mask_spans(8, 1, causal=False, prefix_lens=torch.ones(1, 1, device=dev, dtype=torch.int32))
    with pytest.raises(ValueError, match="doc_starts"):
        mask_spans(8, 2, doc_starts=torch.zeros(1, 3, device=dev, dtype=torch.int32))
    with pytest.raises(TypeError, match="doc_starts"):
        mask_spans(8, 1, doc_starts=torch.zeros(1, 3, device=dev))


def test_more_rows_than_keys(dev):
    """With intervals and no bias, where the rows sit is not read; else it has to be said."""
    from ssa_amd import masked_attention

    q, k, v, dout = _inputs(14, BF16, 1, 90, 20, 4, 2, 64)
    spans = torch.stack((torch.arange(90) % 20, torch.arange(90) % 20 + 1 + torch.arange(90) // 30), 1).clamp(max=20).int()
    res = _run(dev, q, k, v, dout, spans[None])
    _check(res, q, k, v, dout, spans[None], 0.0, None, 0)
    with pytest.raises(RuntimeError, match="q_pos0"):
        masked_attention(q.to(dev), k.to(dev), v.to(dev))
    with pytest.raises(RuntimeError, match="q_pos0"):
        masked_attention(q.to(dev), k.to(dev), v.to(dev), spans[None].to(dev), slopes=_slopes(4).to(dev))


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64), (BF16, 128)], ids=str)
def test_far_rows(dev, dtype, d):
    """Rows of q, k, v and dout 16 MiB apart: offsets past 2^31 elements and 2^32 bytes."""
    from ssa_amd import masked_attention

    n, h_q, h_kv = 300, 4, 2
    q, k, v, dout = _inputs(15, dtype, 1, n, n, h_q, h_kv, d)
    step = (16 << 20) // q.element_size()
    pool = torch.zeros((n - 1) * step + 32 * d, device=dev, dtype=dtype)
    at, far = 0, []
    for t in (q, k, v, dout):
        x = torch.as_strided(pool, t.shape, (0, step, d, 1), at)
        x.copy_(t)
        far.append(x)
        at += t.shape[2] * d
    assert (n - 1) * step * q.element_size() > 1 << 32
    leaves = [t.detach().requires_grad_(True) for t in far[:3]]
    out = masked_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, far[3])
    res = dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))
    _check(res, q, k, v, dout, spans_of(n, n, 0)[None], 0.0, None, 0)


@pytest.mark.parametrize("dtype,d,g", [(F32, 64, 1), (BF16, 64, 4), (BF16, 128, 16)], ids=str)
def test_far_heads(dev, dtype, d, g):
    """Heads of q, k, v and dout 16 MiB apart, 144 of them: offsets past 2^31 bytes of a row."""
    from ssa_amd import masked_attention

    n, h_q = 70, 144
    q, k, v, dout = _inputs(16, dtype, 1, n, n, h_q, h_q // g, d)
    step = (16 << 20) // q.element_size()
    pool = torch.zeros((h_q - 1) * step + 4 * n * d, device=dev, dtype=dtype)
    assert (h_q - 1) * step * q.element_size() > 1 << 31
    far = []
    for i, t in enumerate((q, k, v, dout)):
        x = torch.as_strided(pool, t.shape, (0, d, step, 1), i * n * d)
        x.copy_(t)
        far.append(x)
    leaves = [t.detach().requires_grad_(True) for t in far[:3]]
    out = masked_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, far[3])
    res = dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))
    _check(res, q, k, v, dout, spans_of(n, n, 0)[None], 0.0, None, 0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("bad", [0.0, math.nan])
def test_distances_past_2_to_the_24(dev, dtype, bad):
    """A few rows and keys behind 2^24 others: the distance between them is exact in the
    gradients as in the output, also where a hidden row's NaN has a key's sums formed pair by pair."""
    from ssa_amd import masked_attention

    far, n_q, n, h_q, h_kv, d = (1 << 24) + 3, 40, 45, 2, 1, 8
    q, k, v, dout = _inputs(18, dtype, 1, n_q, n, h_q, h_kv, d)
    spans = spans_of(n, n_q, n - n_q, starts=[0, 30, n])
    spans[3] = 0
    if bad != bad:
        q[0, 3], dout[0, 3] = bad, bad
    slopes = torch.tensor([1.0, 0.5])
    pool = torch.zeros(2, 1, far + n, h_kv, d, device=dev, dtype=dtype)
    pool[0, :, far:], pool[1, :, far:] = k.to(dev), v.to(dev)
    leaves = [t.detach().requires_grad_(True) for t in (q.to(dev), pool[0], pool[1])]
    moved = torch.where(spans[:, 1:] > 0, spans + far, spans)[None].to(dev)
    out = masked_attention(*leaves, moved, slopes=slopes.to(dev))
    dq, dk, dv = torch.autograd.grad(out, leaves, dout.to(dev))
    assert not dk[:, :far].any() and not dv[:, :far].any()
    res = {"out": out, "dq": dq, "dk": dk[:, far:], "dv": dv[:, far:]}
    _check(res, q, k, v, dout, spans[None], 0.0, slopes, n - n_q)


@pytest.mark.parametrize("dtype,d,h_q,g,apart", [(F32, 64, 6, 2, 40), (BF16, 128, 8, 4, 100), (BF16, 64, 32, 16, 160)], ids=str)
def test_heads_of_long_sequences(dev, dtype, d, h_q, g, apart):
    """Heads ``apart`` MiB from each other, as views [B, n, h, d] of [B, h, n, d] have them past
    65536 tokens; in the last case a group's heads lie further apart than the backward reads them."""
    from ssa_amd import masked_attention

    n = 70
    q, k, v, dout = _inputs(19, dtype, 1, n, n, h_q, h_q // g, d)
    step = (apart << 20) // q.element_size()
    pool = torch.zeros((h_q - 1) * step + 4 * n * d, device=dev, dtype=dtype)
    far = []
    for i, t in enumerate((q, k, v, dout)):
        x = torch.as_strided(pool, t.shape, (0, d, step, 1), i * n * d)
        x.copy_(t)
        far.append(x)
    leaves = [t.detach().requires_grad_(True) for t in far[:3]]
    out = masked_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, far[3])
    res = dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))
    _check(res, q, k, v, dout, spans_of(n, n, 0)[None], 0.0, None, 0)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64), (BF16, 128)], ids=str)
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_rows_without_keys_beside_hidden_values(dev, dtype, d, cap):
    """Rows that see nothing are zeros also where they share a tile with rows that see keys, and
    that tile holds hidden values that are not finite.  Few heads and many: waves that share
    rows, and that do not; few rows over many keys: parts."""
    for h_kv, n, n_q in ((2, 150, 150), (270, 150, 150), (2, 1600, 21)):
        q, k, v, dout = _inputs(21, dtype, 1, n_q, n, 2 * h_kv, h_kv, d)
        p0 = n - n_q
        spans = spans_of(n, n_q, p0, starts=[0, n - n_q // 2])
        dead = spans[:, 0] == spans[:, 1]
        k[0, n - n_q // 2:], v[0, n - n_q // 2:] = math.nan, math.inf
        q[0, dead], dout[0, dead] = math.inf, math.nan
        res = _run(dev, q, k, v, dout, spans[None], cap)
        assert dead.any() and not dead.all()
        assert (res["out"].cpu()[0, dead] == 0).all() and (res["dq"].cpu()[0, dead] == 0).all()
        few = slice(0, 4), slice(0, 2)
        want = attend(q[0, :, few[0]], k[0, :, few[1]], v[0, :, few[1]], spans, cap, None, p0, dout[0, :, few[0]])
        for name, (value, bound) in want.items():
            check(res[name][0, :, few[0 if name in ("out", "dq") else 1]], value, bound, f"{name}, {h_kv} heads")


def test_tangents_are_refused(dev):
    """Forward-mode differentiation, which a raw call would pass by."""
    import torch.autograd.forward_ad as fwd
    from ssa_amd import masked_attention, sparse_exact_attention

    q, k, v, _ = (t.to(dev) for t in _inputs(22, F32, 1, 8, 8, 4, 2, 16))
    idx = torch.zeros(1, 8, 2, 4, device=dev, dtype=torch.int64)
    want = masked_attention(q, k, v)
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: masked_attention(dual, k, v), lambda: sparse_exact_attention(dual, k, v, idx)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(masked_attention(q, k, v), want)


def test_backward_from_views_of_the_output(dev):
    """kernels.masked_attention_backward with out and out_low as strided views, one of them off alignment."""
    from ssa_amd import kernels

    q, k, v, dout = (t.to(dev) for t in _inputs(23, BF16, 1, 50, 50, 4, 2, 64))
    out, low, lse = kernels.masked_attention(q, k, v, with_lse=True)
    want = kernels.masked_attention_backward(q, k, v, out, dout, lse, out_low=low)
    for first, second in ((4, 8), (8, 4)):
        o, l = (torch.nn.functional.pad(t, (at, 16 - at))[..., at:at + 64] for t, at in ((out, first), (low, second)))
        assert o.stride() == l.stride() and (o.data_ptr() % 16 != 0) != (l.data_ptr() % 16 != 0)
        got = kernels.masked_attention_backward(q, k, v, o, dout, lse, out_low=l)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_mask_spans_of_64_bit_bounds(dev):
    """Starts and prefixes of int64 that 32 bits do not hold stay past every key."""
    from ssa_amd import mask_spans

    n = 20
    starts = torch.tensor([[0, 5, 1 << 32], [3, 1 << 33, (1 << 63) - 1]], device=dev)
    got = mask_spans(n, 2, doc_starts=starts, prefix_lens=torch.tensor([[1 << 32, 0], [(1 << 62) + 7, 0]], device=dev)).cpu()
    assert torch.equal(got[0], spans_of(n, n, 0, starts=[0, 5, n], prefix=[n, 0]))
    assert torch.equal(got[1], spans_of(n, n, 0, starts=[3, n, n], prefix=[n, 0]))
    whole = mask_spans(n, 2, causal=False, doc_starts=starts).cpu()
    assert torch.equal(whole[0], spans_of(n, n, 0, False, starts=[0, 5, n])) and torch.equal(whole[1], spans_of(n, n, 0, False, starts=[3, n, n]))
