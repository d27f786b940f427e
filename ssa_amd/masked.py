"""Dense attention whose rows each see one or two intervals of keys, with capped scores and a
distance bias, forward and backward on HIP kernels.

``dense_attention`` (ssa/attention.py:118-158) takes an ``[n, n]`` bool mask and forms
all n x n scores.  The masks of packed, prefixed and causal sequences are an interval
of keys per row, two behind a sliding window with first keys that stay visible, which is what ``masked_attention`` takes: nothing of size n x n exists,
and keys that no row of a tile sees are not read.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib, kernels


def mask_spans(seq_len: int, batch: int = 1, *, causal: bool = True, doc_starts: Optional[torch.Tensor] = None,
               prefix_lens: Optional[torch.Tensor] = None, num_queries: Optional[int] = None,
               q_pos0: Optional[int] = None, device=None, window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """Key interval [lo, hi) of every row for ``masked_attention``: int32 [batch, num_queries, 2],
    or with ``window`` two of them: [batch, num_queries, 4].

    ``causal``: keys up to the row's own position, else all.  ``doc_starts`` (int [batch,
    documents + 1], ascending) packs documents: document x is the keys ``doc_starts[b, x]``
    to ``doc_starts[b, x + 1]``, rows see their own document only, and rows outside every
    document (padding) see nothing.  Sequences with fewer documents repeat their last start.
    ``prefix_lens`` (int [batch, documents]) opens each document with that many keys that all
    its rows see, whatever their position (an image before its text).  With ``num_queries``
    rows fewer than keys, row i sits at key position ``q_pos0 + i`` (default: the last ones).
    ``window`` w (with causal rows) leaves a row the w keys up to its own, and the first
    ``sinks`` keys of its document (up to its own; of a prefix all).

    Made once for a batch, it serves every layer's forward and backward."""
    n_q = seq_len if num_queries is None else num_queries
    if q_pos0 is None:
        q_pos0 = seq_len - n_q
    if prefix_lens is not None and not causal:
        raise ValueError("prefix_lens goes with causal=True: without it every row sees its whole document")
    if window is not None and (window < 1 or not causal):
        raise ValueError(f"window must be positive and goes with causal=True, got window={window}")
    if sinks < 0 or (sinks > 0 and window is None):
        raise ValueError(f"sinks must not be negative and go with a window, got sinks={sinks}, window={window}")
    if device is None:
        device = next((t.device for t in (doc_starts, prefix_lens) if t is not None), torch.device("cuda"))
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError(f"ssa_amd runs on AMD GPUs (HIP); got device '{device}'.")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if prefix_lens is not None and prefix_lens.dim() == 1 and doc_starts is None:
        prefix_lens = prefix_lens[:, None]
    return kernels.mask_spans(seq_len, batch, n_q, q_pos0, causal, doc_starts, prefix_lens, device,
                              0 if window is None else min(int(window), 1 << 31), min(int(sinks), 1 << 31))


class _MaskedAttention(torch.autograd.Function):
    """ssa_masked_attention with ssa_masked_attention_backward; spans and slopes get no gradient."""

    @staticmethod
    def forward(ctx, q, k, v, spans, scale, softcap, slopes, q_pos0):
        out, low, lse = kernels.masked_attention(q, k, v, spans, scale, softcap, slopes, q_pos0, with_lse=True)
        ctx.save_for_backward(q, k, v, out, low, lse, spans, slopes)
        ctx.rule = (scale, softcap, q_pos0)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, low, lse, spans, slopes = ctx.saved_tensors
        scale, softcap, q_pos0 = ctx.rule
        dq, dk, dv = kernels.masked_attention_backward(q, k, v, out, dout, lse, spans, scale, softcap, slopes, q_pos0,
                                                       low)
        return dq, dk, dv, None, None, None, None, None


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, spans: Optional[torch.Tensor] = None, *,
                     scale: Optional[float] = None, softcap: Optional[float] = None,
                     slopes: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None) -> torch.Tensor:
    """softmax(scores) . v over each row's keys; ``[B, n_q, h_q, d]`` (or ``[n_q, h_q, d]``).

    ``q [B, n_q, h_q, d]``, ``k, v [B, n, h_kv, d]`` (query head j uses KV head
    ``j // (h_q // h_kv)``; unbatched shapes too); ``spans`` from ``mask_spans`` or any int32
    ``[B, n_q, 2]`` of key intervals [lo, hi), or ``[B, n_q, 4]`` of two each (lo, hi, lo2, hi2,
    in any order; a key in both counts once), None for causal.  Scores are q.k / scale
    (sqrt(d)); ``softcap`` c makes them c tanh(s / c); ``slopes`` (float32 [h_q]) subtracts
    slopes[h] |position - key|, row i at position ``q_pos0 + i`` (default n - n_q).  Slopes
    get no gradient.

    Rows that see no key are zeros, and keys a row does not see have no influence on it,
    whatever they hold.  float32 and bfloat16, head_dim a multiple of 8 up to 128; float16
    is widened to float32.  Differentiable in q, k and v; repeated calls give the same bits."""
    _lib.refuse_tangents("masked_attention", q, k, v, slopes)
    unbatched = q.dim() == 3
    if unbatched:
        q, k, v = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
        if spans is not None and spans.dim() == 2:
            spans = spans.unsqueeze(0)
    out_dtype = q.dtype
    if q.dtype == torch.float16:
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
        q, k, v = q.float(), k.float(), v.float()
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("slopes get no gradient: detach them")
    args = (q, k, v, spans, scale, softcap or 0.0)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _MaskedAttention.apply(*args, slopes, q_pos0)
    else:
        out = kernels.masked_attention(*args, slopes, q_pos0)
    if out.dtype != out_dtype:
        out = out.to(out_dtype)
    return out[0] if unbatched else out
