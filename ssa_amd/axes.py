"""Rotary positions with several axes (time, height, width) for images and video.

``apply_rope`` and ``rope_rows`` turn every feature pair by one position; here each pair
belongs to one axis and turns by the token's position on it.  Text tokens, whose
positions are the same on every axis, turn as with one axis.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib, kernels


def axis_rope_freqs(rot: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """Turning speeds of the rot / 2 feature pairs, float64: ``theta ** (-2m / rot)``."""
    return theta ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)


class _RopeAxes(torch.autograd.Function):
    """ssa_rope_axes with its transpose (the turn back) as the backward, to any order."""

    @staticmethod
    def forward(ctx, q, k, plan, positions, freqs, inverse):
        ctx.save_for_backward(positions, freqs)  # (the plan reads them: they must be as they were)
        ctx.plan, ctx.inverse = plan, inverse
        q, k = kernels.axes_run(plan, q, k, inverse)
        return q if k is None else (q, k)

    @staticmethod
    def backward(ctx, dq, dk=None):
        ctx.saved_tensors
        plan, inverse = ctx.plan, not ctx.inverse
        if torch.is_grad_enabled():
            out = _RopeAxes.apply(dq, dk, plan, plan.positions, plan.freqs, inverse)
            dq, dk = (out, None) if dk is None else out
        else:
            dq, dk = kernels.axes_run(plan, dq, dk, inverse)
        return dq, dk, None, None, None, None


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
              sections: Sequence[int]):
    """q ``[B, n, h_q, d]`` and k ``[B, n, h_kv, d]`` turned by their tokens' positions.

    ``positions`` int32 or int64 ``[axes, B, n]`` (or ``[axes, n]`` for every sequence),
    ``freqs`` float64 [rot / 2] (``axis_rope_freqs``), ``sections`` the number of feature
    pairs of each axis, rot / 2 in all: pair m is features (m, m + rot / 2), the first
    ``sections[0]`` pairs turn by ``positions[0]``, the next by ``positions[1]``, ...;
    features from rot on pass through.  Returns (q, k), or q alone when k is None, in their
    dtype; shapes without B are kept.  Angles are exact for far positions (64 bits), the
    result is rounded once.  Differentiable in q and k, not in freqs."""
    _lib.refuse_tangents("rope_axes", q, k, freqs)
    unbatched = q.dim() == 3
    if unbatched:
        q, k = q.unsqueeze(0), None if k is None else k.unsqueeze(0)
    if freqs.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("freqs get no gradient: detach them")
    half = q.dtype == torch.float16
    if half:
        if k is not None and k.dtype != q.dtype:
            raise ValueError(f"k must have q's dtype {q.dtype}, got {k.dtype}")
        q, k = q.float(), None if k is None else k.float()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _RopeAxes.apply(q, k, kernels.axes_plan(q, k, positions, freqs, sections), positions, freqs, False)
        out = (out,) if k is None else out
    else:
        out = kernels.rope_axes(q, k, positions, freqs, sections)
    if half:
        out = tuple(None if x is None else x.half() for x in out)
    if unbatched:
        out = tuple(None if x is None else x[0] for x in out)
    return out[0] if k is None else out
