"""The kernels that the long and wide calls of masked_attention and paged_step run, at sizes
that just reach them, against the 64-bit oracle (tests/dense_oracle.py) on the first and the
last KV head.  tests/test_dense_cuts.py holds the cut of every case here, so that a rule that
moves does not take a kernel out of reach unnoticed."""

import math

import pytest
import torch

from tests.dense_oracle import attend, check, spans_of
from tests.test_gpu_paged import _batch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16

# dtype, B, n, n_q, h_kv, g, d -> forward: waves that share rows, parts of the keys; backward: waves
# that share rows (dQ), groups of 32 keys of a block and parts of the rows (dK, dV)
MASKED = [
    ((BF16, 2, 600, 600, 14, 4, 64), (1, 1, 2, 4, 9)),     # 532 row blocks
    ((BF16, 2, 600, 600, 11, 4, 64), (1, 1, 2, 4, 11)),    # 418: the tiles' order folds
    ((BF16, 2, 600, 600, 11, 4, 128), (1, 1, 2, 4, 6)),
    ((BF16, 1, 600, 600, 12, 4, 64), (2, 1, 2, 4, 18)),    # 228
    ((BF16, 1, 600, 600, 12, 4, 128), (2, 1, 2, 4, 10)),
    ((BF16, 1, 4200, 700, 5, 4, 128), (1, 4, 4, 4, 4)),    # parts, joined
    ((BF16, 2, 600, 600, 27, 4, 64), (1, 1, 1, 4, 4)),     # 1026
    ((BF16, 2, 601, 601, 27, 4, 128), (1, 1, 1, 4, 3)),
    ((BF16, 4, 301, 301, 45, 2, 128), (1, 1, 2, 4, 1)),    # dK, dV in one part: blocks suffice
    ((BF16, 2, 301, 301, 172, 2, 64), (1, 1, 1, 4, 1)),
    ((BF16, 2, 301, 301, 15, 1, 64), (4, 1, 4, 2, 2)),
    ((BF16, 2, 1101, 1101, 9, 4, 64), (1, 1, 2, 4, 7)),    # more than 64 row tiles
    ((BF16, 2, 1101, 1101, 9, 4, 80), (1, 1, 2, 4, 4)),
    ((F32, 2, 600, 600, 11, 4, 64), (1, 1, 2, 4, 6)),
    ((F32, 2, 601, 601, 27, 4, 64), (1, 1, 1, 4, 3)),
    ((F32, 2, 600, 600, 9, 4, 64), (2, 1, 2, 4, 7)),
    ((F32, 1, 601, 601, 12, 4, 128), (2, 1, 2, 4, 10)),
    ((F32, 2, 600, 600, 14, 4, 96), (1, 1, 2, 4, 5)),
    ((F32, 2, 600, 600, 27, 4, 128), (1, 1, 1, 4, 3)),
    ((F32, 2, 301, 301, 86, 2, 64), (1, 1, 2, 4, 1)),
    ((F32, 2, 301, 301, 15, 1, 64), (4, 1, 4, 2, 2)),
]

# dtype, sequences (new, cached), h_kv, g, d -> waves that share rows, parts of the keys;
# whether the call's own rows are a third of the longest sequence's keys or more
PAGED = [
    ((BF16, [(500, 700), (420, 3), (80, 64)], 13, 4, 64), (1, 1), True),
    ((BF16, [(500, 700), (420, 3), (80, 64)], 13, 4, 128), (1, 1), True),
    ((BF16, [(500, 1700), (420, 3), (80, 640)], 13, 4, 64), (1, 1), False),
    ((BF16, [(500, 1700), (420, 3), (80, 640)], 13, 4, 128), (1, 1), False),
    ((BF16, [(400, 600), (300, 33), (200, 0)], 7, 4, 64), (2, 1), True),
    ((BF16, [(400, 600), (300, 33), (200, 0)], 7, 4, 128), (2, 1), True),
    ((BF16, [(400, 1600), (300, 33), (200, 0)], 7, 4, 64), (2, 1), False),
    ((BF16, [(400, 1600), (300, 33), (200, 0)], 7, 4, 96), (2, 1), False),
    ((F32, [(500, 700), (420, 3), (80, 64)], 13, 4, 64), (1, 1), True),
    ((F32, [(500, 700), (420, 3), (80, 64)], 13, 4, 128), (1, 1), True),
    ((F32, [(500, 1700), (420, 3), (80, 640)], 13, 4, 64), (1, 1), False),
    ((F32, [(500, 1700), (420, 3), (80, 640)], 13, 4, 128), (1, 1), False),
    ((F32, [(400, 600), (300, 33), (200, 0)], 9, 4, 64), (2, 1), True),
    ((F32, [(400, 600), (300, 33), (200, 0)], 9, 4, 128), (2, 1), True),
    ((F32, [(400, 1600), (300, 33), (200, 0)], 9, 4, 64), (2, 1), False),
    ((F32, [(400, 1600), (300, 33), (200, 0)], 9, 4, 128), (2, 1), False),
    ((BF16, [(300, 4700), (100, 31), (1, 900)], 4, 7, 128), (1, 8), False),
    ((F32, [(300, 4700), (100, 31), (1, 900)], 4, 7, 64), (1, 8), False),
]


def _slopes(h_q):
    return torch.tensor([2.0 ** (-4.0 * (i + 1) / h_q) for i in range(h_q)])


@pytest.mark.parametrize("rule", ["plain", "cap", "bias"])
@pytest.mark.parametrize("case", [c for c, _ in MASKED], ids=str)
def test_masked(dev, case, rule):
    """Causal; documents with capped scores, NaN and infinities in the padding behind them; and
    prefixes with capped scores and a distance bias."""
    from ssa_amd import mask_spans, masked_attention

    dtype, B, n, n_q, h_kv, g, d = case
    h_q, p0 = h_kv * g, n - n_q
    gen = torch.Generator().manual_seed(71)
    q, k, v, dout = (torch.randn(B, m, h, d, generator=gen).to(dtype) for m, h in ((n_q, h_q), (n, h_kv), (n, h_kv), (n_q, h_q)))
    cap, slopes = {"plain": 0.0, "cap": 3.0, "bias": 4.0}[rule], _slopes(h_q) if rule == "bias" else None
    if rule == "plain":
        spans, dev_spans = [spans_of(n, n_q, p0)] * B, None
    else:
        end = n - 45
        starts = [[0, n // 6, n // 6, n // 2, end] if b % 2 else [n // 9, n // 3, end - 1, end, end] for b in range(B)]
        prefix = [[(s[i + 1] - s[i]) // 2 + i for i in range(4)] for s in starts] if rule == "bias" else None
        spans = [spans_of(n, n_q, p0, True, starts[b], prefix[b] if prefix else None) for b in range(B)]
        dev_spans = mask_spans(n, B, doc_starts=torch.tensor(starts, device=dev), num_queries=n_q,
                               prefix_lens=None if prefix is None else torch.tensor(prefix, device=dev))
        assert torch.equal(dev_spans.cpu(), torch.stack(spans)), "mask_spans"
    if rule == "cap":
        k[:, end:], v[:, end:] = math.nan, math.inf
        for b in range(B):
            dead = spans[b][:, 0] == spans[b][:, 1]
            q[b, dead], dout[b, dead] = math.inf, math.nan
    print(f"masked {rule} {case}", flush=True)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = masked_attention(*leaves, dev_spans, softcap=cap or None, slopes=None if slopes is None else slopes.to(dev))
    res = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout.to(dev)))))
    for b, kv in ((0, 0), (B - 1, h_kv - 1)):
        of, mine = slice(kv * g, (kv + 1) * g), slice(kv, kv + 1)
        want = attend(q[b, :, of], k[b, :, mine], v[b, :, mine], spans[b], cap, None if slopes is None else slopes[of], p0,
                      dout[b, :, of])
        for name, (value, bound) in want.items():
            check(res[name][b, :, of if name in ("out", "dq") else mine], value, bound, f"{name}[{b}], KV head {kv}")


@pytest.mark.parametrize("rule", ["plain", "cap", "bias"])
@pytest.mark.parametrize("case", [c for c, _, _ in PAGED], ids=str)
def test_paged(dev, case, rule):
    """_batch leaves NaN in the pages' rows that hold no key, so the last tile's sums are formed again."""
    from ssa_amd import paged_step

    dtype, seqs, h_kv, g, d = case
    h_q, page = h_kv * g, 16
    cap, slopes = {"plain": 0.0, "cap": 3.0, "bias": 4.0}[rule], _slopes(h_q) if rule == "bias" else None
    s, keys = _batch(72, dtype, seqs, h_q, h_kv, d, page)
    print(f"paged {rule} {case}", flush=True)
    out = paged_step(**{n: t.to(dev) for n, t in s.items()}, softcap=cap or None, slopes=None if slopes is None else slopes.to(dev),
                     max_new=max(m for m, _ in seqs), max_len=max(m + c for m, c in seqs), check=True)
    for kv in (0, h_kv - 1):
        at, of, mine = 0, slice(kv * g, (kv + 1) * g), slice(kv, kv + 1)
        for b, (m, c) in enumerate(seqs):
            want = attend(s["q"][at:at + m, of], *(t[:, mine] for t in keys[b]), spans_of(c + m, m, c), cap,
                          None if slopes is None else slopes[of], c)["out"]
            check(out[at:at + m, of], *want, f"sequence {b}, KV head {kv}")
            at += m


# Sums formed again go key by key, without rounding weights to bf16, in another order.  fp32: two scores
# of d products are (d + 8) 2^-24 sum |q k| / sqrt(d) apart at most, the sum about 0.64 sqrt(d)
# (128: 6e-5), twice for the weight's and the sum's, from both sides: 2^-12 of the largest value.
# bf16: a weight's rounding (2^-8 of the values' mean) and the outputs' on both sides.
TIGHT = {F32: 2.0 ** -12, BF16: 2.0 ** -7}


@pytest.mark.parametrize("case", [c for c, _ in MASKED], ids=str)
def test_masked_values_of_later_tokens(dev, case):
    """A key near the end whose scores and values are not finite: the rows before it, whose tiles hold
    it, are as they were, and the rows behind it are not finite."""
    from ssa_amd import masked_attention

    dtype, B, n, n_q, h_kv, g, d = case
    gen = torch.Generator().manual_seed(73)
    q, k, v = (torch.randn(B, m, h, d, generator=gen).to(dtype).to(dev) for m, h in ((n_q, h_kv * g), (n, h_kv), (n, h_kv)))
    print(f"masked {case}", flush=True)
    want = masked_attention(q, k, v)
    at = n - 7
    k[:, at], v[:, at] = math.nan, math.inf
    out = masked_attention(q, k, v)
    row = at - (n - n_q)
    assert torch.isfinite(out[:, :row]).all() and not torch.isfinite(out[:, row:]).any()
    assert ((out[:, :row].float() - want[:, :row].float()).abs() <= TIGHT[dtype] * (want[:, :row].float().abs() + v.float().abs().nan_to_num(posinf=0).amax())).all()


@pytest.mark.parametrize("case", [c for c, _, _ in PAGED], ids=str)
def test_paged_values_of_later_tokens(dev, case):
    """The same of a chunk's last token: its row alone is not finite."""
    from ssa_amd import paged_step

    dtype, seqs, h_kv, g, d = case
    s, _ = _batch(74, dtype, seqs, h_kv * g, h_kv, d, 16)
    x = {n: t.to(dev) for n, t in s.items()}
    kw = dict(max_new=max(m for m, _ in seqs), max_len=max(m + c for m, c in seqs))
    print(f"paged {case}", flush=True)
    want = paged_step(**x, **kw)
    last = [int(e) - 1 for e, (m, _) in zip(s["starts"][1:], seqs) if m > 1]
    for i in last:
        x["k"][i], x["v"][i] = math.nan, math.inf
    out = paged_step(**x, **kw)
    bad = torch.zeros(out.shape[0], dtype=torch.bool, device=dev)
    bad[last] = True
    assert not torch.isfinite(out[bad]).any() and torch.isfinite(out[~bad]).all()
    most = max(float(t.float().nan_to_num(posinf=0, neginf=0).abs().max()) for t in (s["v"], s["v_pages"]))
    assert ((out[~bad].float() - want[~bad].float()).abs() <= TIGHT[dtype] * (want[~bad].float().abs() + most)).all()
