"""Attention of rows that see any set of keys in 64 bits, with its gradients and how far a
kernel may be from each value; what windows, trees and pages of 8 bits stand for.

The bounds count the roundings that the kernels make, as tests/dense_oracle.py's do (u = 2^-24
a term of an fp32 sum; r = 2^-8, half a step of bf16, for each weight or score gradient that
enters a product, for the output that D = dO . o is formed from and for the result).  A scale
of a key or value multiplies a score or a weight in fp32: one more u each, and the weight is
rounded after it."""

from __future__ import annotations

import math
import random

import torch

U = 2.0 ** -24
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def attend_set(q, k, v, see, qpos, kpos, cap=0.0, slopes=None, dout=None, r=None):
    """q [m, h_q, d], k, v [n, h_kv, d], see bool [m, n], positions qpos [m] and kpos [n].
    Returns {"out": (value, bound), ...}, with dq, dk and dv too where dout is given."""
    if r is None:
        r = 0.0 if q.dtype == torch.float32 else 2.0 ** -8
    m, h_q, d = q.shape
    n, h_kv = k.shape[0], k.shape[1]
    g, scale = h_q // h_kv, math.sqrt(d)
    q, k, v = q.double(), k.double(), v.double()
    used, live = see.any(0), see.any(1)   # what nothing visible touches may hold anything
    zero = lambda *s: [torch.zeros(*s, dtype=torch.float64) for _ in range(2)]  # noqa: E731
    res = {"out": zero(m, h_q, d)}
    if dout is not None:
        res.update(dq=zero(m, h_q, d), dk=zero(n, h_kv, d), dv=zero(n, h_kv, d))
    for h in range(h_q):
        kh, vh = (torch.where(used[:, None], x[:, h // g], 0.0) for x in (k, v))
        qh = torch.where(live[:, None], q[:, h], 0.0)
        raw, mag = qh @ kh.T / scale, qh.abs() @ kh.abs().T / scale
        err = (d + 10) * U * mag + 4 * U * raw.abs()
        t = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
        s = cap * t if cap else raw
        if cap:
            err = err + cap * 2.0 ** -21
        if slopes is not None:
            far = (qpos[:, None] - kpos[None]).abs().double()
            s = s - float(slopes[h]) * far
            err = err + 8 * U * float(slopes[h]) * far
        err = err + 8 * U * s.abs() + 8 * U
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(1, keepdim=True)
        p = torch.where(see, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        worst = torch.where(see, err, 0.0).amax(1, keepdim=True)
        rel = torch.where(see, 2 * worst + 2 * err + (n + 10) * U, 0.0)
        o = p @ vh
        b = (p * (2 * rel + r)) @ vh.abs() + (n + 10) * U * (p @ vh.abs())
        ob = b + r * (o.abs() + b) + 1e-30
        res["out"][0][:, h], res["out"][1][:, h] = o, ob
        if dout is None:
            continue
        do = torch.where(live[:, None], dout.double()[:, h], 0.0)
        dp = do @ vh.T
        dsum = (do * o).sum(1, keepdim=True)
        dp_err = (d + 8) * U * (do.abs() @ vh.abs().T)
        dsum_err = (do.abs() * ob).sum(1, keepdim=True) + (d + 8) * U * (do.abs() * o.abs()).sum(1, keepdim=True)
        f = 1.0 - t * t
        ds, mags = p * (dp - dsum) * f / scale, p * (dp.abs() + dsum.abs()) / scale
        b = mags * (2 * rel + 8 * U) + p * (dp_err + dsum_err) / scale
        if cap:  # 1 - t^2 is formed from a tanh that is off by 2^-21
            b = b + mags * 2.0 ** -19
        e = ds.abs() * r + (1 + r) * b
        dq = ds @ kh
        b = e @ kh.abs() + (n + 8) * U * (ds.abs() @ kh.abs())
        res["dq"][0][:, h], res["dq"][1][:, h] = dq, b + r * (dq.abs() + b) + 1e-30
        res["dk"][0][:, h // g] += ds.T @ qh
        res["dk"][1][:, h // g] += e.T @ qh.abs() + (m * g + 8) * U * (ds.abs().T @ qh.abs())
        res["dv"][0][:, h // g] += p.T @ do
        res["dv"][1][:, h // g] += (p * (2 * rel + r)).T @ do.abs() + (m * g + 8) * U * (p.T @ do.abs())
    for x in ("dk", "dv"):
        if x in res:
            val, b = res[x]
            res[x][1] = b + r * (val.abs() + b) + 1e-30
    return {x: tuple(y) for x, y in res.items()}


def held(x, dtype):
    """Rows x [..., d] as codes of dtype and float32 scales, from the definition in 64 bits."""
    x = x.double()
    most = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    scale = torch.where(most < 2.0 ** -100, 0.0, most / MOST[dtype]).float()
    y = torch.where((fine & (scale > 0))[..., None], x / scale.double().clamp(min=1e-300)[..., None], 0.0)
    if dtype == torch.int8:
        codes = y.round().to(torch.int8)
    else:  # multiples of 2^-9 up to 2^-6, from there on eight a factor of two
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
        codes = ((y / step).round() * step).float().to(dtype)
    return codes, torch.where(fine, scale, math.nan)


def values(codes, scale):
    return codes.float().double() * scale.double()[..., None]


def tree(m, r: random.Random, flat=0.7):
    """Parents of m drafts; flat: large for bushy trees."""
    return [max(-1, i - 1 - int(r.expovariate(flat))) for i in range(m)]


def sees(m, cached, parents=None, window=0, sinks=0):
    """(see [m, cached + m], qpos, kpos) of a sequence's new tokens, row by row from the definition."""
    n = cached + m
    see = torch.zeros(m, n, dtype=torch.bool)
    qpos, kpos = torch.arange(cached, n), torch.arange(n)
    for i in range(m):
        family = list(range(i + 1))
        if parents is not None:
            family, at = [], i
            while at >= 0:
                family.append(at)
                at = parents[at]
        qpos[i] = cached + len(family) - 1
        kpos[cached + i] = qpos[i]
        see[i, :cached] = True
        see[i, [cached + x for x in family]] = True
    if window:
        see &= (qpos[:, None] - kpos[None] < window) | (kpos[None] < sinks)
    return see, qpos, kpos
