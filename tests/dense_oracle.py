"""Dense attention with a key interval per row in 64 bits, with its gradients, and how far
a kernel may be from each value.

The bounds follow from the roundings that the kernels make: fp32 products and sums
(u = 2^-24 a term), scores exact up to those, and for bf16 tensors one rounding
(r = 2^-8, half a step) of each weight or score gradient that enters a product, of the
output that D = dO . o is formed from, and of the result."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def spans_of(n, n_q, q_pos0, causal=True, starts=None, prefix=None):
    """Key intervals [n_q, 2] of one sequence, row by row from the definition."""
    rows = []
    for i in range(n_q):
        pos, lo, end, pre = q_pos0 + i, 0, n, 0
        if starts is not None:
            inside = [x for x in range(len(starts) - 1) if starts[x] <= pos < starts[x + 1]]
            if not inside:
                rows.append((0, 0))
                continue
            lo, end = starts[inside[0]], min(starts[inside[0] + 1], n)
            pre = prefix[inside[0]] if prefix is not None else 0
        elif prefix is not None:
            pre = prefix[0]
        hi = min(max(pos + 1, lo + pre), end) if causal else end
        rows.append((lo, hi) if hi > lo else (0, 0))
    return torch.tensor(rows, dtype=torch.int32).reshape(n_q, 2)


def attend(q, k, v, spans, cap=0.0, slopes=None, q_pos0=0, dout=None, scale=None, round_to=None, cap_rel=None):
    """One sequence: q [m, h_q, d], k, v [n, h_kv, d] (any dtype), spans [m, 2].  Returns
    {"out": (value, bound), ...} with dq, dk and dv too where dout is given.  ``cap_rel``: how
    far a capped score may be off relative to itself, in place of cap 2^-21."""
    r = 0.0 if (round_to or q.dtype) == torch.float32 else 2.0 ** -8
    m, h_q, d = q.shape
    n, h_kv = k.shape[0], k.shape[1]
    g = h_q // h_kv
    scale = math.sqrt(d) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    zero = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    res = {"out": [zero(m, h_q, d), zero(m, h_q, d)]}
    if dout is not None:
        dout = dout.double()
        res.update(dq=[zero(m, h_q, d), zero(m, h_q, d)], dk=[zero(n, h_kv, d), zero(n, h_kv, d)],
                   dv=[zero(n, h_kv, d), zero(n, h_kv, d)])
    j = torch.arange(n)
    pos = q_pos0 + torch.arange(m)
    see = (j[None] >= spans[:, :1]) & (j[None] < spans[:, 1:])
    for h in range(h_q):
        qh, kh, vh = q[:, h], k[:, h // g], v[:, h // g]
        # keys and rows that nothing visible touches may hold anything
        used = see.any(0)
        kh, vh = torch.where(used[:, None], kh, 0.0), torch.where(used[:, None], vh, 0.0)
        live = see.any(1)
        qh = torch.where(live[:, None], qh, 0.0)
        raw = qh @ kh.T / scale
        mag = qh.abs() @ kh.abs().T / scale
        ds_bound = (d + 8) * U * mag + 4 * U * raw.abs()     # error of a score
        t = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
        s = cap * t if cap else raw
        if cap:
            ds_bound = ds_bound + (cap * 2.0 ** -21 if cap_rel is None else cap_rel * s.abs())
        if slopes is not None:
            far = (pos[:, None] - j[None]).abs().double()
            s = s - float(slopes[h]) * far
            ds_bound = ds_bound + 8 * U * float(slopes[h]) * far
        ds_bound = ds_bound + 8 * U * s.abs() + 8 * U
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(1, keepdim=True)
        w = torch.where(see, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
        p = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        # relative error of a weight: its score's and the largest score's, the sum's
        worst = torch.where(see, ds_bound, 0.0).amax(1, keepdim=True)
        rel = 2 * worst + 2 * ds_bound + (n + 8) * U
        rel = torch.where(see, rel, 0.0)
        o = p @ vh
        res["out"][0][:, h] = o
        o_bound = (p * (2 * rel + r)) @ vh.abs() + (n + 8) * U * (p @ vh.abs())
        res["out"][1][:, h] = o_bound + r * (o.abs() + o_bound) + 1e-30
        if dout is None:
            continue
        do = torch.where(live[:, None], dout[:, h], 0.0)
        dp = do @ vh.T
        dsum = (do * o).sum(1, keepdim=True)
        dp_bound = (d + 8) * U * (do.abs() @ vh.abs().T)
        dsum_bound = (do.abs() * res["out"][1][:, h]).sum(1, keepdim=True) + (d + 8) * U * (do.abs() * o.abs()).sum(1, keepdim=True)
        f = 1.0 - t * t
        ds = p * (dp - dsum) * f / scale
        mags = p * (dp.abs() + dsum.abs()) / scale
        b = mags * (2 * rel + 8 * U) + p * (dp_bound + dsum_bound) / scale
        if cap:  # 1 - t^2 is formed from a tanh that is off by 2^-21
            b = b + mags * 2.0 ** -19
        e = ds.abs() * r + (1 + r) * b
        dq = ds @ kh
        res["dq"][0][:, h] = dq
        b = e @ kh.abs() + (n + 8) * U * (ds.abs() @ kh.abs())
        res["dq"][1][:, h] = b + r * (dq.abs() + b) + 1e-30
        res["dk"][0][:, h // g] += ds.T @ qh
        res["dk"][1][:, h // g] += e.T @ qh.abs() + (m * g + 8) * U * (ds.abs().T @ qh.abs())
        res["dv"][0][:, h // g] += p.T @ do
        res["dv"][1][:, h // g] += (p * (2 * rel + r)).T @ do.abs() + (m * g + 8) * U * (p.T @ do.abs())
    for x in ("dk", "dv"):
        if x in res:
            val, b = res[x]
            res[x][1] = b + r * (val.abs() + b) + 1e-30
    return {x: tuple(y) for x, y in res.items()}


def check(got, want, bound, what):
    """Every value of got within bound of want."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: values that are not finite"
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert over.max() <= 0, (f"{what}: off by {float((got - want).abs().flatten()[at]):.3e} where "
                             f"{float(bound.flatten()[at]):.3e} is allowed (value {float(want.flatten()[at]):.3e}, index {at})")
