"""Tensor-level wrappers over the libssa_hip entry points (one per C-ABI call).

All sequence tensors are batched ``[B, n, heads, d]`` views whose last
dimension is contiguous; other strides are passed through, so transposed
layouts such as HF's ``[B, heads, n, d]`` (permuted) need no copy.  Outputs and
workspaces come from the PyTorch caching allocator on the input's device, and
every call is enqueued on the current stream without synchronising.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import call, ptr, stream_of


def _check_rows(x: torch.Tensor, name: str) -> None:
    if x.dim() != 4:
        raise ValueError(f"{name} must be [B, n, heads, d], got shape {tuple(x.shape)}")
    if x.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


def _f32c(t: torch.Tensor) -> torch.Tensor:
    return t.detach().to(torch.float32).contiguous()


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, rot: int, by_head: bool,
         inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of ``x`` [B, n, h, d] (ssa_rope): features j < rot rotate in
    pairs (j, j + rot/2) as ``x * cos + rotate_half(x) * sin``; the rest pass through.

    ``cos``/``sin`` are ``[rows, >= rot]`` (one table) or ``[B, rows, >= rot]``
    with a contiguous last dimension; the angle row is the head index
    (``by_head``, SSAAttention's apply_rope call) or the token position (Hugging
    Face).  ``inverse`` applies the transpose (the gradient).  ``out`` defaults
    to a new contiguous tensor of x's dtype; ``out is x`` rotates in place."""
    _check_rows(x, "x")
    _lib.require_device(x, cos, sin)
    B, n, h, d = x.shape
    if cos.shape != sin.shape or cos.dtype != sin.dtype:
        raise ValueError("cos and sin tables must have the same shape and dtype")
    if cos.stride(-1) != 1 or sin.stride(-1) != 1 or cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    if cos.dim() == 2:
        t_sb, t_sr, rows = 0, cos.stride(0), cos.shape[0]
    elif cos.dim() == 3 and cos.shape[0] in (1, B):
        t_sb = cos.stride(0) if cos.shape[0] == B else 0
        t_sr, rows = cos.stride(1), cos.shape[1]
    else:
        raise ValueError(f"rope tables must be [rows, w] or [B, rows, w], got {tuple(cos.shape)}")
    if cos.shape[-1] < rot:
        raise ValueError(f"rope tables are {cos.shape[-1]} wide, rot={rot} needs that many")
    if out is None:
        out = torch.empty((B, n, h, d), device=x.device, dtype=x.dtype)
    call("ssa_rope", ptr(x), _lib.elem_dtype(x), B, n, h, d, x.stride(0), x.stride(1), x.stride(2),
         ptr(cos), ptr(sin), _lib.elem_dtype(cos), t_sb, t_sr, rows, int(rot),
         _lib.ROPE_BY_HEAD if by_head else _lib.ROPE_BY_POSITION, int(bool(inverse)),
         ptr(out), _lib.elem_dtype(out), out.stride(0), out.stride(1), out.stride(2), stream_of(x))
    return out


def route_vectors(x: torch.Tensor, w: torch.Tensor, group: int) -> torch.Tensor:
    """normalize(mean_g(x . w^T)) -> float32 [B, heads/group, n, d_s] (ssa/router.py:102-117)."""
    _check_rows(x, "x")
    _lib.require_device(x, w)
    B, n, h_in, d = x.shape
    w = _f32c(w)
    d_s = w.shape[0]
    out = torch.empty((B, h_in // group, n, d_s), device=x.device, dtype=torch.float32)
    call("ssa_route_vectors", ptr(x), _lib.elem_dtype(x), B, n, h_in, group, d,
         x.stride(0), x.stride(1), x.stride(2), ptr(w), d_s, ptr(out), stream_of(x))
    return out


def normalize_rows(x: torch.Tensor) -> torch.Tensor:
    """Row-wise F.normalize of a float32 matrix (ssa/router.py:118)."""
    _lib.require_device(x)
    x = _f32c(x)
    out = torch.empty_like(x)
    d_s = x.shape[-1]
    call("ssa_normalize_rows", ptr(x), x.numel() // d_s, d_s, ptr(out), stream_of(x))
    return out


def code_topk(xhat: torch.Tensor, chat: torch.Tensor, top: int,
              temperature: float = 1.0, exhaustive: bool = False) -> torch.Tensor:
    """Top-`top` codes per row, int32 [B, h, rows, top] (ssa/router.py:121-130,141).

    ``exhaustive=True`` skips the matrix-core screen and scores every code in
    fp32 (same result; used to cross-check the screen)."""
    _lib.require_device(xhat, chat)
    xhat = xhat.contiguous()
    chat = chat.contiguous()
    B, h, rows, d_s = xhat.shape
    n_c = chat.shape[1]
    codes = torch.empty((B, h, rows, top), device=xhat.device, dtype=torch.int32)
    ws, ws_bytes = None, 0
    if not exhaustive:
        ws_bytes = int(_lib.load().ssa_code_topk_workspace_bytes(B, h, rows, n_c))
        ws = torch.empty(max(ws_bytes, 1), device=xhat.device, dtype=torch.uint8)
    call("ssa_code_topk", ptr(xhat), B, h, rows, ptr(chat), n_c, d_s, float(temperature), top,
         ptr(codes), ptr(ws), ws_bytes, stream_of(xhat))
    return codes


def route_codes(q: torch.Tensor, k: torch.Tensor, w_qr: torch.Tensor, w_kr: torch.Tensor,
                codebook: torch.Tensor, a: int, b: int,
                temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Stage (a): (q_codes int32 [B,h_kv,n,a], k_codes int32 [B,h_kv,n,b])."""
    _check_rows(q, "q")
    _check_rows(k, "k")
    _lib.require_device(q, k, w_qr, w_kr, codebook)
    if q.dtype != k.dtype:
        raise TypeError(f"q and k must share a dtype ({q.dtype} vs {k.dtype})")
    B, n, h_q, d = q.shape
    h_kv = k.shape[2]
    w_qr, w_kr, codebook = _f32c(w_qr), _f32c(w_kr), _f32c(codebook)
    n_c, d_s = codebook.shape[1], codebook.shape[2]
    dev = q.device
    q_codes = torch.empty((B, h_kv, n, a), device=dev, dtype=torch.int32)
    k_codes = torch.empty((B, h_kv, n, b), device=dev, dtype=torch.int32)
    ws_bytes = _lib.load().ssa_route_workspace_bytes(B, n, h_kv, n_c, d_s)
    ws = torch.empty(max(int(ws_bytes), 1), device=dev, dtype=torch.uint8)
    call("ssa_route_codes", ptr(q), ptr(k), _lib.elem_dtype(q), B, n, h_q, h_kv, d,
         q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
         ptr(w_qr), ptr(w_kr), ptr(codebook), d_s, n_c, a, b, float(temperature),
         ptr(q_codes), ptr(k_codes), ptr(ws), ws_bytes, stream_of(q))
    return q_codes, k_codes


def build_index(k_codes: torch.Tensor, n_c: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Stage (b): offsets int32 [B,h,n_c+1], postings int32 [B,h,n*b] (ascending per bucket)."""
    _lib.require_device(k_codes)
    k_codes = k_codes.contiguous()
    B, h, n, b = k_codes.shape
    dev = k_codes.device
    offsets = torch.empty((B, h, n_c + 1), device=dev, dtype=torch.int32)
    postings = torch.empty((B, h, n * b), device=dev, dtype=torch.int32)
    ws_bytes = _lib.load().ssa_index_workspace_bytes(B, n, h, b, n_c)
    ws = torch.empty(max(int(ws_bytes), 1), device=dev, dtype=torch.uint8)
    call("ssa_build_index", ptr(k_codes), B, n, h, b, n_c, ptr(offsets), ptr(postings), ptr(ws),
         ws_bytes, stream_of(k_codes))
    return offsets, postings


def query_order(q_codes: torch.Tensor, n_c: int) -> torch.Tensor:
    """Query positions per (batch, kv head) sorted stably by their smallest code
    ``q_codes.min(-1)``: int32 [B, h, n], a processing order for sparse_attention
    (rows sharing that code share its bucket's keys)."""
    _lib.require_device(q_codes)
    q_codes = q_codes.contiguous()
    B, h, n, a = q_codes.shape
    order = torch.empty((B, h, n), device=q_codes.device, dtype=torch.int32)
    ws_bytes = _lib.load().ssa_query_order_workspace_bytes(B, n, h, n_c)
    ws = torch.empty(max(int(ws_bytes), 1), device=q_codes.device, dtype=torch.uint8)
    call("ssa_query_order", ptr(q_codes), B, n, h, a, n_c, ptr(order), ptr(ws), ws_bytes,
         stream_of(q_codes))
    return order


def select(q: torch.Tensor, k: torch.Tensor, q_codes: torch.Tensor, offsets: torch.Tensor,
           postings: torch.Tensor, b: int, top_k: int, mask_mode: int = _lib.MASK_CAUSAL,
           mask: Optional[torch.Tensor] = None, score_div: Optional[float] = None,
           index_dtype: torch.dtype = torch.int64,
           with_stats: bool = False, sorted: bool = True, use_workspace: Union[bool, int] = True,
           row_order: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None,
           row_prefix: Optional[torch.Tensor] = None):
    """Stage (c): candidate indices [B, n_q, h_kv, top_k] (ssa/router.py:151-214).

    ``q`` and ``q_codes`` may hold fewer rows (n_q) than ``k`` has keys (n): a
    block of queries at key positions ``q_pos0 .. q_pos0 + n_q - 1`` (default:
    the last n_q positions, as in decoding against a cache).  With n_q = n this
    is the whole sequence.

    ``mask`` (MASK_DENSE) is a bool/uint8 ``[n, n]`` or ``[B, n, n]`` tensor with a
    contiguous last dimension.  ``with_stats`` also returns int32 ``[B, h_kv, n, 2]``
    (unique candidates, postings read inside the mask window) per row.
    ``sorted=False`` lists the same selected set in ascending index order (then
    the same filler).  ``use_workspace=False`` runs the one-block-per-row kernel
    for every row; an int gives the workspace size in bytes instead of the
    recommended ``ssa_select_workspace_bytes(B, n, h_kv, top_k)`` (same results).
    ``row_order`` (int32 [B, h_kv, n], a permutation of 0..n-1 per head, e.g.
    ``query_order``) only sets the order in which rows are processed.
    ``row_prefix`` (int32 [B, h_kv, n_q], written): X per row, the key prefix
    [0, X) its indices hold exactly once (the lowest-key filler), for
    ``sparse_attention``'s dense-prefix pass.
    """
    _check_rows(q, "q")
    _check_rows(k, "k")
    _lib.require_device(q, k, q_codes, offsets, postings, mask)
    B, n_q, h_q, d = q.shape
    n = k.shape[1]
    if q_pos0 is None:
        q_pos0 = n - n_q
    h_kv = k.shape[2]
    a = q_codes.shape[-1]
    n_c = offsets.shape[-1] - 1
    q_codes, offsets, postings = q_codes.contiguous(), offsets.contiguous(), postings.contiguous()
    if score_div is None:
        score_div = float(torch.tensor(d ** 0.5, dtype=torch.float32))
    m_sb = m_si = 0
    if mask_mode == _lib.MASK_DENSE:
        if mask is None:
            raise ValueError("MASK_DENSE needs a mask tensor")
        if mask.dtype == torch.bool:
            mask = mask.view(torch.uint8)
        if mask.stride(-1) != 1:
            mask = mask.contiguous()
        if mask.dim() == 2:
            m_sb, m_si = 0, mask.stride(0)
        else:
            m_sb, m_si = mask.stride(0), mask.stride(1)
    if row_order is not None:
        _lib.require_device(row_order)
        if row_order.dtype != torch.int32 or tuple(row_order.shape) != (B, h_kv, n_q):
            raise ValueError(f"row_order must be int32 [{B}, {h_kv}, {n_q}]")
        row_order = row_order.contiguous()
    if row_prefix is not None:
        _lib.require_device(row_prefix)
        if (row_prefix.dtype != torch.int32 or tuple(row_prefix.shape) != (B, h_kv, n_q)
                or not row_prefix.is_contiguous()):
            raise ValueError(f"row_prefix must be a contiguous int32 [{B}, {h_kv}, {n_q}] tensor")
    out = torch.empty((B, n_q, h_kv, top_k), device=q.device, dtype=index_dtype)
    stats = torch.empty((B, h_kv, n_q, 2), device=q.device, dtype=torch.int32) if with_stats else None
    ws_bytes, ws = 0, None
    if use_workspace is True:
        ws_bytes = int(_lib.load().ssa_select_workspace_bytes(B, n_q, h_kv, top_k))
    elif use_workspace is not False:
        ws_bytes = int(use_workspace)
    if ws_bytes > 0:
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8)
    call("ssa_select_block", ptr(q), ptr(k), _lib.elem_dtype(q), B, n, n_q, q_pos0, h_q, h_kv, d,
         q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
         ptr(q_codes), a, ptr(offsets), ptr(postings), n_c, b, top_k, mask_mode, ptr(mask),
         m_sb, m_si, float(score_div), int(bool(sorted)), ptr(row_order), ptr(out), _lib.index_dtype(out),
         ptr(stats), ptr(row_prefix), ptr(ws), ws_bytes, stream_of(q))
    return (out, stats) if with_stats else out


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, idx: torch.Tensor,
                     scale_div: Optional[float] = None, causal: bool = False,
                     out: Optional[torch.Tensor] = None,
                     error_flag: Optional[torch.Tensor] = None,
                     row_order: Optional[torch.Tensor] = None,
                     q_pos0: Optional[int] = None, dense_prefix: bool = True,
                     row_prefix: Optional[torch.Tensor] = None,
                     row_stats: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stage (d): gathered exact attention, [B, n_q, h_q, d] in q's dtype (ssa/attention.py:12-115).

    ``row_order`` (int32 [B, h_kv, n_q], a permutation of 0..n_q-1 per head) only
    sets the order in which rows are processed; results are the same.  ``q`` and
    ``idx`` may hold fewer rows (n_q) than ``k``/``v`` have keys: query row r
    then sits at key position ``q_pos0 + r`` (default n - n_q), which is what
    ``causal`` compares the indices with.  ``dense_prefix`` (bf16, d 64 or 128):
    the keys [0, X) a row's indices hold exactly once are attended in blocks of
    neighbouring rows that load them once (a workspace of the library's size);
    ``row_prefix`` (int32 [B, h_kv, n_q], from ``select``) gives X per row, which
    the pass otherwise finds from the indices."""
    for name, t in (("q", q), ("k", k), ("v", v), ("indices", idx)):
        _check_rows(t, name)
    _lib.require_device(q, k, v, idx)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    B, n_q, h_q, d = q.shape
    n = k.shape[1]
    if q_pos0 is None:
        q_pos0 = n - n_q
    h_kv = k.shape[2]
    top_k = idx.shape[-1]
    if scale_div is None:
        scale_div = math.sqrt(d)
    if out is None:
        out = torch.empty((B, n_q, h_q, d), device=q.device, dtype=q.dtype)
    if row_order is not None:
        _lib.require_device(row_order)
        if row_order.dtype != torch.int32 or tuple(row_order.shape) != (B, h_kv, n_q):
            raise ValueError(f"row_order must be int32 [{B}, {h_kv}, {n_q}]")
        row_order = row_order.contiguous()
    ws_bytes = 0
    if dense_prefix:
        ws_bytes = int(_lib.load().ssa_sparse_attention_workspace_bytes(
            _lib.elem_dtype(q), B, n_q, h_q, h_kv, d, top_k))
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    if row_prefix is not None:
        _lib.require_device(row_prefix)
        if (row_prefix.dtype != torch.int32 or tuple(row_prefix.shape) != (B, h_kv, n_q)
                or not row_prefix.is_contiguous()):
            raise ValueError(f"row_prefix must be a contiguous int32 [{B}, {h_kv}, {n_q}] tensor")
    _check_stats(row_stats, B, h_kv, n_q, h_q)
    call("ssa_sparse_attention_block", ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), B, n, n_q, q_pos0,
         h_q, h_kv, d,
         q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
         v.stride(0), v.stride(1), v.stride(2), ptr(idx), _lib.index_dtype(idx), top_k,
         idx.stride(0), idx.stride(1), idx.stride(2), float(scale_div), int(bool(causal)),
         ptr(row_order), ptr(row_prefix), ptr(out), _lib.elem_dtype(out), out.stride(0), out.stride(1),
         out.stride(2), ptr(error_flag), ptr(row_stats), ptr(ws), ws_bytes, stream_of(q))
    return out


def _check_stats(row_stats, B, h_kv, n, h_q):
    if row_stats is None:
        return
    _lib.require_device(row_stats)
    if (row_stats.dtype != torch.float32 or tuple(row_stats.shape) != (B, h_kv, n, h_q // h_kv, 2)
            or not row_stats.is_contiguous()):
        raise ValueError(f"row_stats must be a contiguous fp32 [{B}, {h_kv}, {n}, {h_q // h_kv}, 2] tensor")


def row_stats_buffer(q: torch.Tensor, h_kv: int) -> torch.Tensor:
    """NaN-filled fp32 [B, h_kv, n, g, 2] for sparse_attention(row_stats=...):
    the matrix-core forward writes each (row, head)'s softmax reference and
    1 / sum, which sparse_attention_backward(row_stats=...) then reuses; entries
    left NaN (other paths) are recomputed by the backward."""
    B, n, h_q = q.shape[0], q.shape[1], q.shape[2]
    return torch.full((B, h_kv, n, h_q // h_kv, 2), float("nan"), device=q.device, dtype=torch.float32)


def block_indices(idx: torch.Tensor, block_size: int, n_k_blocks: Optional[int] = None,
                  error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Key blocks per query block, int64 [B, ceil(n / block_size), h_kv, n_k_blocks]
    (ssa/triton_kernel.py:226-294) from token selections ``idx`` [B, n, h_kv, top_k];
    n_k_blocks defaults to min(top_k, number of blocks).  Ranked by reference
    count, then lower block id."""
    _check_rows(idx, "indices")
    _lib.require_device(idx)
    B, n, h_kv, top_k = idx.shape
    nb = (n + block_size - 1) // block_size
    if n_k_blocks is None:
        n_k_blocks = min(top_k, nb)
    out = torch.empty((B, nb, h_kv, n_k_blocks), device=idx.device, dtype=torch.int64)
    call("ssa_block_indices", ptr(idx), _lib.index_dtype(idx), B, n, h_kv, top_k,
         idx.stride(0), idx.stride(1), idx.stride(2), int(block_size), int(n_k_blocks), ptr(out),
         _lib.index_dtype(out), out.stride(0), out.stride(1), out.stride(2), ptr(error_flag),
         stream_of(idx))
    return out


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor,
                           block_size: int, scale_div: Optional[float] = None,
                           out: Optional[torch.Tensor] = None,
                           error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal exact attention of each query over the key blocks listed for its
    query block: ``blocks`` [B, ceil(n / block_size), h_kv, n_k_blocks]
    (ssa/triton_kernel.py:141-223, with an exact normalised softmax)."""
    for name, t in (("q", q), ("k", k), ("v", v), ("block_indices", blocks)):
        _check_rows(t, name)
    _lib.require_device(q, k, v, blocks)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    B, n, h_q, d = q.shape
    h_kv = k.shape[2]
    nb = (n + block_size - 1) // block_size
    if tuple(blocks.shape[:3]) != (B, nb, h_kv):
        raise ValueError(f"block_indices must be [{B}, {nb}, {h_kv}, n_k_blocks], got {tuple(blocks.shape)}")
    if scale_div is None:
        scale_div = math.sqrt(d)
    if out is None:
        out = torch.empty((B, n, h_q, d), device=q.device, dtype=q.dtype)
    call("ssa_block_sparse_attention", ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), B, n, h_q, h_kv, d,
         q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
         v.stride(0), v.stride(1), v.stride(2), ptr(blocks), _lib.index_dtype(blocks),
         int(block_size), blocks.shape[-1], blocks.stride(0), blocks.stride(1), blocks.stride(2),
         float(scale_div), ptr(out), _lib.elem_dtype(out), out.stride(0), out.stride(1), out.stride(2),
         ptr(error_flag), stream_of(q))
    return out


class Routing(NamedTuple):
    """What one selection was made from, for the bucket-mode backward: the
    stage (a) codes, the stage (b) key index and whether the selection's mask
    was causal (else none; an explicit mask has no bucket mode)."""
    q_codes: torch.Tensor   # int32 [B, h_kv, n, a]
    k_codes: torch.Tensor   # int32 [B, h_kv, n, b]
    offsets: torch.Tensor   # int32 [B, h_kv, N_c + 1]
    postings: torch.Tensor  # int32 [B, h_kv, n * b]
    causal: bool


def sparse_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, idx: torch.Tensor,
                              out: torch.Tensor, dout: torch.Tensor,
                              scale_div: Optional[float] = None, causal: bool = False,
                              error_flag: Optional[torch.Tensor] = None,
                              row_order: Optional[torch.Tensor] = None,
                              row_prefix: Optional[torch.Tensor] = None,
                              routing: Optional[Routing] = None, bitmap_rows: int = -1,
                              row_stats: Optional[torch.Tensor] = None
                              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of stage (d) w.r.t. q, k, v (fp32, shapes of q, k, v), given the
    forward output ``out`` and its gradient ``dout`` (the autograd backward of
    ssa/attention.py:64-113).

    With ``row_prefix`` and ``routing`` (the selection that produced ``idx``,
    n >= top_k) the candidate slots' dk and dv come from the bucket pass
    (ssa_sparse_attention_backward_routed); ``bitmap_rows`` sizes its key
    bitmaps for rows without filler (-1: half the rows).  ``row_stats``
    (``row_stats_buffer`` filled by the forward) saves the row kernel's first
    pass for the rows it covers.  Same results."""
    for name, t in (("q", q), ("k", k), ("v", v), ("indices", idx), ("out", out), ("dout", dout)):
        _check_rows(t, name)
    _lib.require_device(q, k, v, idx, out, dout)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    B, n, h_q, d = q.shape
    h_kv = k.shape[2]
    top_k = idx.shape[-1]
    if tuple(out.shape) != (B, n, h_q, d) or tuple(dout.shape) != (B, n, h_q, d):
        raise ValueError("out and dout must have q's shape")
    if scale_div is None:
        scale_div = math.sqrt(d)
    dq = torch.zeros((B, n, h_q, d), device=q.device, dtype=torch.float32)
    dk = torch.empty((B, n, h_kv, d), device=q.device, dtype=torch.float32)
    dv = torch.empty((B, n, h_kv, d), device=q.device, dtype=torch.float32)
    if row_order is not None:
        _lib.require_device(row_order)
        if row_order.dtype != torch.int32 or tuple(row_order.shape) != (B, h_kv, n):
            raise ValueError(f"row_order must be int32 [{B}, {h_kv}, {n}]")
        row_order = row_order.contiguous()
    ws_bytes, ws = 0, None
    if row_prefix is not None:
        _lib.require_device(row_prefix)
        if (row_prefix.dtype != torch.int32 or tuple(row_prefix.shape) != (B, h_kv, n)
                or not row_prefix.is_contiguous()):
            raise ValueError(f"row_prefix must be a contiguous int32 [{B}, {h_kv}, {n}] tensor")
        if routing is None:
            ws_bytes = int(_lib.load().ssa_sparse_attention_backward_workspace_bytes(
                _lib.elem_dtype(q), _lib.elem_dtype(dout), B, n, h_q, h_kv, d))
    _check_stats(row_stats, B, h_kv, n, h_q)
    common = (ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), B, n, h_q,
              h_kv, d, q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
              v.stride(0), v.stride(1), v.stride(2), ptr(idx), _lib.index_dtype(idx), top_k,
              idx.stride(0), idx.stride(1), idx.stride(2), float(scale_div), int(bool(causal)),
              ptr(row_order), ptr(out), _lib.elem_dtype(out), out.stride(0), out.stride(1),
              out.stride(2), ptr(dout), _lib.elem_dtype(dout), dout.stride(0), dout.stride(1),
              dout.stride(2), ptr(dq), ptr(dk), ptr(dv), ptr(error_flag), ptr(row_prefix), ptr(row_stats))
    if row_prefix is not None and routing is not None:
        qc, kc, off, post = (_contig_i32(t, name) for t, name in (
            (routing.q_codes, "q_codes"), (routing.k_codes, "k_codes"), (routing.offsets, "offsets"),
            (routing.postings, "postings")))
        _lib.require_device(qc, kc, off, post)
        a, b, n_c = qc.shape[-1], kc.shape[-1], off.shape[-1] - 1
        if (tuple(qc.shape[:3]) != (B, h_kv, n) or tuple(kc.shape[:3]) != (B, h_kv, n)
                or tuple(off.shape[:2]) != (B, h_kv) or tuple(post.shape) != (B, h_kv, n * b)):
            raise ValueError("routing tensors do not match q, k (see kernels.Routing)")
        ws_bytes = int(_lib.load().ssa_sparse_attention_backward_routed_workspace_bytes(
            _lib.elem_dtype(q), _lib.elem_dtype(dout), B, n, h_q, h_kv, d, top_k, a, b, n_c, int(bitmap_rows)))
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
        call("ssa_sparse_attention_backward_routed", *common, ptr(qc), a, ptr(kc), b, ptr(off), ptr(post),
             n_c, int(bool(routing.causal)), ptr(ws), ws_bytes, stream_of(q))
        return dq, dk, dv
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    call("ssa_sparse_attention_backward", *common, ptr(ws), ws_bytes, stream_of(q))
    return dq, dk, dv


def _contig_i32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    return t if t.is_contiguous() else t.contiguous()


# ---- dense attention with key intervals, paged cache, axes -------------------
# A call of these on small tensors takes about as long on the host as on the GPU:
# raw addresses and the raw stream go to the library, contiguous tensors skip the
# stride checks, and workspace sizes (functions of the sizes alone) are remembered.


def _on_device(first: torch.Tensor, *rest: Optional[torch.Tensor]) -> int:
    """The HIP device all of these tensors are on."""
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            _lib.require_device(first, *rest)
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    if dev < 0:
        _lib.require_device(first)
    return dev


def _call_on(dev: int, name: str, *args) -> None:
    """``call`` on the current stream of device ``dev``, with it current (launches go to the
    current device)."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch._C._cuda_getDevice():
        call(name, *args, stream)
    else:
        with torch.cuda.device(dev):
            call(name, *args, stream)


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows16(t: torch.Tensor):
    """(t, its element strides but the last one), t's rows contiguous and aligned to 16 bytes: a
    contiguous copy where they are not.  A dimension of one element does not step."""
    e = t.element_size()
    if not t.is_contiguous():
        st = tuple(0 if x == 1 else s for s, x in zip(t.stride(), t.shape))
        if (st[-1] == 1 or t.shape[-1] == 1) and not any(s * e % 16 for s in st[:-1]) and t.data_ptr() % 16 == 0:
            return t, st[:-1]
        t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    if t.dim() == 4:
        _, n, h, d = t.shape
        return t, (n * h * d, h * d, d)
    _, h, d = t.shape
    return t, (h * d, d)


def _group_rows16(t: torch.Tensor, g: int):
    """``_rows16`` of q or dout [B, n, heads, d] for the backward, which wants the heads of a group
    of g within 2 GiB: a contiguous copy where they lie further apart."""
    t, st = _rows16(t)
    _, _, h, d = t.shape
    if ((126 + g) // g * st[1] + (g - 1) * st[2] + d) * t.element_size() > 0x7FFFFFF0:
        n = t.shape[1]
        return t.contiguous(), (n * h * d, h * d, d)
    return t, st


@functools.lru_cache(maxsize=1024)
def _bytes(name: str, *sizes) -> int:
    return int(getattr(_lib.load(), name)(*sizes))


def _workspace(nbytes: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, device=like.device, dtype=torch.uint8) if nbytes else None


def _once(t: torch.Tensor, name: str) -> None:
    """Refuses a tensor to write to whose elements share memory (an expanded one)."""
    if not t.is_contiguous() and any(s == 0 and x > 1 for s, x in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} is written to, but some of its elements are the same memory")


def _check_slopes(slopes: Optional[torch.Tensor], h_q: int) -> Optional[torch.Tensor]:
    if slopes is None:
        return None
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (h_q,):
        raise ValueError(f"slopes must be float32 [{h_q}]")
    return slopes.contiguous()


def _pos0(q_pos0: Optional[int], n: int, n_q: int, spans, slopes) -> int:
    """Position of query row 0; where neither mask nor bias reads it, any will do."""
    if q_pos0 is not None:
        return q_pos0
    return n - n_q if n >= n_q or spans is None or slopes is not None else 0


def mask_spans(n: int, batch: int, n_q: int, q_pos0: int, causal: bool, doc_starts: Optional[torch.Tensor],
               prefix_lens: Optional[torch.Tensor], device: torch.device) -> torch.Tensor:
    """Key interval of each row, int32 [batch, n_q, 2] (ssa_mask_spans)."""
    out = torch.empty((batch, n_q, 2), device=device, dtype=torch.int32)
    dev = _on_device(out, doc_starts, prefix_lens)
    docs = 1 if doc_starts is None else doc_starts.shape[-1] - 1
    if doc_starts is not None:
        if doc_starts.dim() != 2 or doc_starts.shape[0] != batch or docs < 1:
            raise ValueError(f"doc_starts must be [{batch}, documents + 1], got {tuple(doc_starts.shape)}")
        doc_starts = _index32(doc_starts, "doc_starts")
    if prefix_lens is not None:
        if tuple(prefix_lens.shape) != (batch, docs):
            raise ValueError(f"prefix_lens must be [{batch}, {docs}], got {tuple(prefix_lens.shape)}")
        prefix_lens = _index32(prefix_lens, "prefix_lens")
    _call_on(dev, "ssa_mask_spans", _at(doc_starts), docs, _at(prefix_lens), batch, n, n_q, q_pos0, int(bool(causal)),
             out.data_ptr())
    return out


def _index32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.dtype == torch.int64:  # (a bound far past the keys stays past them)
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(torch.int32).contiguous()


def _check_dense(q, k, v, spans):
    """(B, n_q, h_q, d, n, h_kv) of matching q, k, v and spans."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, n, heads, d], got shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    B, n_q, h_q, d = q.shape
    _, n, h_kv, _ = k.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != d:
        raise ValueError(f"k and v must be [{B}, n, h_kv, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if h_kv == 0 or h_q % h_kv != 0:
        raise ValueError(f"{h_q} query heads are not divisible by {h_kv} KV heads")
    if spans is not None and (spans.dtype != torch.int32 or tuple(spans.shape) != (B, n_q, 2) or not spans.is_contiguous()):
        raise ValueError(f"spans must be a contiguous int32 [{B}, {n_q}, 2] tensor")
    return B, n_q, h_q, d, n, h_kv


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, spans: Optional[torch.Tensor] = None,
                     scale_div: Optional[float] = None, softcap: float = 0.0,
                     slopes: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None, with_lse: bool = False):
    """Dense attention over each row's key interval (ssa_masked_attention): [B, n_q, h_q, d]
    in q's dtype.  ``with_lse`` returns (out, out_low, lse) for the backward: what rounding left of a
    bf16 output (None for float32) and the float32 [B, h_q, n_q] log2 sums.
    ``spans`` None: causal.  Query row i sits at key position ``q_pos0 + i`` (default n - n_q)."""
    dev = _on_device(q, k, v, spans, slopes)
    B, n_q, h_q, d, n, h_kv = _check_dense(q, k, v, spans)
    slopes = _check_slopes(slopes, h_q)
    q, qs = _rows16(q)
    k, ks = _rows16(k)
    v, vs = _rows16(v)
    dt = _lib.elem_dtype(q)
    out = torch.empty((B, n_q, h_q, d), device=q.device, dtype=q.dtype)
    low = lse = None
    if with_lse:
        lse = torch.empty((B, h_q, n_q), device=q.device, dtype=torch.float32)
        low = torch.empty_like(out) if dt == _lib.DTYPE_BF16 else None
    nbytes = _bytes("ssa_masked_attention_workspace_bytes", dt, B, n, n_q, h_q, h_kv, d)
    ws = _workspace(nbytes, q)
    _call_on(dev, "ssa_masked_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, B, n, n_q,
             _pos0(q_pos0, n, n_q, spans, slopes), h_q, h_kv, d, *qs, *ks, *vs, _at(spans),
             math.sqrt(d) if scale_div is None else scale_div, softcap, _at(slopes), out.data_ptr(), n_q * h_q * d, h_q * d, d,
             _at(low), _at(lse), _at(ws), nbytes)
    return (out, low, lse) if with_lse else out


def masked_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, dout: torch.Tensor,
                              lse: torch.Tensor, spans: Optional[torch.Tensor] = None, scale_div: Optional[float] = None,
                              softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None,
                              out_low: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of masked_attention w.r.t. q, k and v, in their dtype and contiguous, from the
    forward's ``out``, ``lse`` and (bf16) ``out_low`` and the output gradient."""
    dev = _on_device(q, k, v, out, dout, lse, spans, slopes, out_low)
    B, n_q, h_q, d, n, h_kv = _check_dense(q, k, v, spans)
    if tuple(out.shape) != (B, n_q, h_q, d) or tuple(dout.shape) != (B, n_q, h_q, d):
        raise ValueError("out and dout must have q's shape")
    if out.dtype != q.dtype or dout.dtype != q.dtype:
        raise TypeError(f"out and dout must have q's dtype {q.dtype}")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, h_q, n_q) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 [{B}, {h_q}, {n_q}] tensor")
    if out_low is not None and (out_low.shape != out.shape or out_low.dtype != out.dtype or out_low.stride() != out.stride()):
        raise ValueError("out_low must have out's shape, strides and dtype")
    slopes = _check_slopes(slopes, h_q)
    dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    q, qs = _group_rows16(q, h_q // h_kv)
    k, ks = _rows16(k)
    v, vs = _rows16(v)
    if out_low is not None and not out.is_contiguous():  # (one may be copied and not the other: they share strides)
        out, out_low = out.contiguous(), out_low.contiguous()
    out, os = _rows16(out)
    dout, dos = _group_rows16(dout, h_q // h_kv)
    out_low = None if out_low is None else _rows16(out_low)[0]
    dt = _lib.elem_dtype(q)
    nbytes = _bytes("ssa_masked_attention_backward_workspace_bytes", dt, B, n, n_q, h_q, h_kv, d)
    ws = _workspace(nbytes, q)
    _call_on(dev, "ssa_masked_attention_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, B, n, n_q,
             _pos0(q_pos0, n, n_q, spans, slopes), h_q, h_kv, d, *qs, *ks, *vs, _at(spans),
             math.sqrt(d) if scale_div is None else scale_div, softcap, _at(slopes), out.data_ptr(), _at(out_low), *os,
             dout.data_ptr(), *dos, lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _at(ws), nbytes)
    return dq, dk, dv


def paged_step(q: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor], k_pages: torch.Tensor,
               v_pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, cached: torch.Tensor,
               scale_div: Optional[float] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
               max_new: Optional[int] = None, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
               error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """New tokens of a ragged batch appended to their pages and attended (ssa_paged_step):
    q [T, h_q, d], k and v [T, h_kv, d] (None: already in the pages), pools
    [pages, page size, h_kv, d], table int32 [B, width], starts int32 [B + 1], cached int32
    [B].  ``max_new`` and ``max_len`` bound a sequence's new tokens and keys (defaults: T and
    what the table holds)."""
    dev = _on_device(q, k, v, k_pages, v_pages, table, starts, cached, slopes, out, error_flag)
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("q must be [T, h_q, d] and the pools [pages, page size, h_kv, d]")
    T, h_q, d = q.shape
    pages, page, h_kv, dp = k_pages.shape
    if dp != d or h_kv == 0 or h_q % h_kv != 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit pages {tuple(k_pages.shape)}")
    dtype = q.dtype
    for name, t in (("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("out", out)):
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{name} must have q's dtype {dtype}, got {t.dtype}")
    B, width = table.shape
    for name, t, shape in (("table", table, (B, width)), ("starts", starts, (B + 1,)), ("cached", cached, (B,))):
        if t.dtype != torch.int32 or t.shape != shape or (shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name} must be an int32 {list(shape)} tensor with contiguous rows")
    pools = []
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        rows, st = _rows16(t) if t.numel() else (t, (0, 0, 0))
        if rows is not t:
            raise ValueError(f"{name} must have contiguous rows aligned to 16 bytes")
        if k is not None:
            _once(t, name)
        pools += st
    slopes = _check_slopes(slopes, h_q)
    if error_flag is not None and (error_flag.dtype != torch.int32 or error_flag.numel() != 1):
        raise ValueError("error_flag must be one int32")
    q, qs = _rows16(q)
    ks = vs = (0, 0)
    if k is not None:
        if k.shape != (T, h_kv, d) or v.shape != (T, h_kv, d):
            raise ValueError(f"k must be [{T}, {h_kv}, {d}] and v too, got {tuple(k.shape)} and {tuple(v.shape)}")
        k, ks = _rows16(k)
        v, vs = _rows16(v)
    name = "ssa_paged_step"
    if out is None:  # (rows that no sequence has, or that are left out, become zeros)
        if B == 0:
            return torch.zeros((T, h_q, d), device=q.device, dtype=dtype)
        name, out = "ssa_paged_step_zeroed", torch.empty((T, h_q, d), device=q.device, dtype=dtype)
    else:
        if out.shape != (T, h_q, d) or _rows16(out)[0] is not out:
            raise ValueError(f"out must be [{T}, {h_q}, {d}] with rows aligned to 16 bytes")
        _once(out, "out")
    max_new = T if max_new is None else min(int(max_new), T)
    max_len = width * page if max_len is None else min(int(max_len), width * page)
    dt = _lib.elem_dtype(q)
    nbytes = _bytes("ssa_paged_step_workspace_bytes", dt, T, B, h_q, h_kv, d, max_new, max_len)
    ws = _workspace(nbytes, q)
    _call_on(dev, name, q.data_ptr(), _at(k), _at(v), dt, T, B, h_q, h_kv, d, *qs, *ks, *vs, k_pages.data_ptr(),
             v_pages.data_ptr(), pages, page, *pools, table.data_ptr(), table.stride(0) if B > 1 else 0, width,
             starts.data_ptr(), cached.data_ptr(), max_new, max_len, math.sqrt(d) if scale_div is None else scale_div,
             softcap, _at(slopes), out.data_ptr(), *_rows16(out)[1], _at(error_flag), _at(ws), nbytes)
    return out


def _steps(t: torch.Tensor):
    """Element strides of [B, n, heads, d] but the last one; a dimension of one element does not step."""
    if t.is_contiguous():
        _, n, h, d = t.shape
        return n * h * d, h * d, d
    return tuple(0 if x == 1 else s for s, x in zip(t.stride()[:-1], t.shape))


class AxesPlan(NamedTuple):
    """What rope_axes turns a (q, k) pair by, checked: the backward's call takes it as it is."""
    dev: int
    dtype: int
    sizes: Tuple[int, ...]     # B, n, h_q, h_k, d
    positions: torch.Tensor
    freqs: torch.Tensor
    turn: tuple                # positions' type and steps, the axes and their sections


def axes_plan(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
              sections) -> AxesPlan:
    """Checks rope_axes' arguments."""
    dev = _on_device(q, k, positions, freqs)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"q and k must be [B, n, heads, d], got {tuple(q.shape)}" + ("" if k is None else f" and {tuple(k.shape)}"))
    B, n, h_q, d = q.shape
    h_k = 0 if k is None else k.shape[2]
    if k is not None and (k.shape != (B, n, h_k, d) or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    axes = len(sections)
    if positions.shape != (axes, B, n) and positions.shape != (axes, n):
        raise ValueError(f"positions must be [{axes}, {B}, {n}] or [{axes}, {n}], got {tuple(positions.shape)}")
    pos_dtype = _lib.index_dtype(positions)
    if n > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("freqs must be float64 [rot / 2] (axis_rope_freqs)")
    freqs = freqs.contiguous()
    return AxesPlan(dev, _lib.elem_dtype(q), (B, n, h_q, h_k, d), positions, freqs,
                    (pos_dtype, positions.stride(0), positions.stride(1) if positions.dim() == 3 else 0, axes,
                     (ctypes.c_int32 * axes)(*sections)))


def axes_run(plan: AxesPlan, q: torch.Tensor, k: Optional[torch.Tensor], inverse: bool
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q and k of the plan's sizes turned (ssa_rope_axes); ``inverse`` applies the transpose.  New
    contiguous tensors of q's dtype."""
    B, n, h_q, h_k, d = plan.sizes
    q = q if q.stride(-1) == 1 else q.contiguous()
    qo = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    k_at, ks, ko, ko_at = None, (0, 0, 0), None, None
    if k is not None:
        k = k if k.stride(-1) == 1 else k.contiguous()
        ko = torch.empty(k.shape, device=q.device, dtype=q.dtype)
        k_at, ks, ko_at = k.data_ptr(), _steps(k), ko.data_ptr()
    _call_on(plan.dev, "ssa_rope_axes", q.data_ptr(), k_at, plan.dtype, B, n, h_q, h_k, d, *_steps(q), *ks,
             plan.positions.data_ptr(), *plan.turn, plan.freqs.data_ptr(), 2 * plan.freqs.shape[0], inverse, qo.data_ptr(),
             n * h_q * d, h_q * d, d, ko_at, n * h_k * d, h_k * d, d)
    return qo, ko


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, sections,
              inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions with several axes on q [B, n, h_q, d] and k [B, n, h_k, d] (or None)
    (ssa_rope_axes): positions int [axes, B, n] or [axes, n], freqs float64 [rot / 2], sections the
    pairs of each axis."""
    return axes_run(axes_plan(q, k, positions, freqs, sections), q, k, inverse)
