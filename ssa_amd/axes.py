"""Rotary positions with several axes (time, height, width) for images and video.

``apply_rope`` and ``rope_rows`` turn every feature pair by one position; here each pair
belongs to one axis and turns by the token's position on it.  Text tokens, whose
positions are the same on every axis, turn as with one axis.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib, kernels


def axis_rope_freqs(rot: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """Turning speeds of the rot / 2 feature pairs, float64: ``theta ** (-2m / rot)``."""
    return theta ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)


class _RopeAxes(torch.autograd.Function):
    """ssa_rope_axes with its transpose (the turn back) as the backward."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, sections):
        ctx.save_for_backward(positions, freqs)
        ctx.sections = sections
        return kernels.rope_axes(q, k, positions, freqs, sections)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, freqs = ctx.saved_tensors
        dq, dk = kernels.rope_axes(dq, dk, positions, freqs, ctx.sections, inverse=True)
        return dq, dk, None, None, None


class _RopeAxesOne(torch.autograd.Function):
    """The same for q alone."""

    @staticmethod
    def forward(ctx, q, positions, freqs, sections):
        ctx.save_for_backward(positions, freqs)
        ctx.sections = sections
        return kernels.rope_axes(q, None, positions, freqs, sections)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dq):
        positions, freqs = ctx.saved_tensors
        return kernels.rope_axes(dq, None, positions, freqs, ctx.sections, inverse=True)[0], None, None, None


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
              sections: Sequence[int]):
    """q ``[B, n, h_q, d]`` and k ``[B, n, h_kv, d]`` turned by their tokens' positions.

    ``positions`` int32 or int64 ``[axes, B, n]`` (or ``[axes, n]`` for every sequence),
    ``freqs`` float64 [rot / 2] (``axis_rope_freqs``), ``sections`` the number of feature
    pairs of each axis, rot / 2 in all: pair m is features (m, m + rot / 2), the first
    ``sections[0]`` pairs turn by ``positions[0]``, the next by ``positions[1]``, ...;
    features from rot on pass through.  Returns (q, k), or q alone when k is None, in their
    dtype; shapes without B are kept.  Angles are exact for far positions (64 bits), the
    result is rounded once.  Differentiable in q and k."""
    unbatched = q.dim() == 3
    if unbatched:
        q, k = q.unsqueeze(0), None if k is None else k.unsqueeze(0)
    _lib.require_device(q, k, positions, freqs)
    if positions.dim() == 2:
        positions = positions[:, None].expand(-1, q.shape[0], -1)
    dtypes = (q.dtype, None if k is None else k.dtype)
    if q.dtype == torch.float16:
        q, k = q.float(), None if k is None else k.float()
    sections = tuple(int(x) for x in sections)
    grad = torch.is_grad_enabled()
    if k is None:
        out = ((_RopeAxesOne.apply(q, positions, freqs, sections) if grad and q.requires_grad
                else kernels.rope_axes(q, None, positions, freqs, sections)[0]),)
    elif grad and (q.requires_grad or k.requires_grad):
        out = _RopeAxes.apply(q, k, positions, freqs, sections)
    else:
        out = kernels.rope_axes(q, k, positions, freqs, sections)
    out = tuple((x[0] if unbatched else x).to(t) for x, t in zip(out, dtypes))
    return out[0] if k is None else out
