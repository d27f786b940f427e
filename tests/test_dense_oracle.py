"""The 64-bit oracle of the dense attention tests against autograd and differences."""

import math

import pytest
import torch

from tests.dense_oracle import attend, spans_of


def _autograd(q, k, v, see, cap, slopes, q_pos0, dout):
    q, k, v = (t.clone().requires_grad_(True) for t in (q, k, v))
    g = q.shape[1] // k.shape[1]
    s = torch.einsum("mhd,nhd->hmn", q, k.repeat_interleave(g, 1)) / math.sqrt(q.shape[2])
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        far = (q_pos0 + torch.arange(q.shape[0])[:, None] - torch.arange(k.shape[0])[None]).abs()
        s = s - slopes.double()[:, None, None] * far
    s = s.masked_fill(~see, -1e30)
    p = torch.softmax(s, -1) * see
    out = torch.einsum("hmn,nhd->mhd", p, v.repeat_interleave(g, 1))
    return (out, *torch.autograd.grad(out, (q, k, v), dout))


@pytest.mark.parametrize("cap,bias,prefix", [(0.0, False, None), (2.0, False, [3, 2]), (0.0, True, None), (3.0, True, [4, 0])])
def test_oracle_against_autograd_and_differences(cap, bias, prefix):
    g = torch.Generator().manual_seed(5)
    m, n, h_q, h_kv, d = 9, 11, 4, 2, 8
    q, k, v, dout = (torch.randn(*s, generator=g, dtype=torch.float64) for s in
                     ((m, h_q, d), (n, h_kv, d), (n, h_kv, d), (m, h_q, d)))
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0]) if bias else None
    spans = spans_of(n, m, 2, starts=[0, 5, 10], prefix=prefix)
    spans[3] = 0  # a row that sees nothing
    see = (torch.arange(n) >= spans[:, :1]) & (torch.arange(n) < spans[:, 1:])
    res = attend(q, k, v, spans, cap, slopes, 2, dout)
    out, dq, dk, dv = _autograd(q, k, v, see, cap, slopes, 2, dout)
    for name, want in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert (res[name][0] - want).abs().max() < 1e-12, name
    assert (res["out"][0][3] == 0).all()
    step = 1e-6
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        way = torch.randn(t.shape, generator=g, dtype=torch.float64)
        ends = []
        for sgn in (1, -1):
            args = {"q": q, "k": k, "v": v}
            args[name[1]] = t + sgn * step * way
            ends.append((attend(args["q"], args["k"], args["v"], spans, cap, slopes, 2)["out"][0] * dout).sum())
        slope = (ends[0] - ends[1]) / (2 * step)
        # central differences: step^2 times a third derivative of order one, and 1e-16 / step
        assert abs(slope - (res[name][0] * way).sum()) < 1e-7 * max(1.0, abs(slope)), name
