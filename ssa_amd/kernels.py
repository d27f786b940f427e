"""Tensor-level wrappers over the libssa_hip entry points (one per C-ABI call).

All sequence tensors are batched ``[B, n, heads, d]`` views whose last
dimension is contiguous; other strides are passed through, so transposed
layouts such as HF's ``[B, heads, n, d]`` (permuted) need no copy.  Outputs and
workspaces come from the PyTorch caching allocator on the input's device, and
every call is enqueued on the current stream without synchronising.
"""

from __future__ import annotations

import ctypes
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


def _call_on(t: torch.Tensor, name: str, *args) -> None:
    """``call`` with t's device current (the launches go to the current device)."""
    if t.device.index == torch.cuda.current_device():
        call(name, *args)
    else:
        with torch.cuda.device(t.device):
            call(name, *args)


def _same_device(**tensors) -> None:
    _lib.require_device(*tensors.values())
    first = next(iter(tensors.values())).device
    for name, t in tensors.items():
        if t is not None and t.device != first:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {first}")


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its rows are not contiguous or not aligned to 16 bytes."""
    e = t.element_size()
    if (t.stride(-1) != 1 and t.shape[-1] > 1) or any(
            s * e % 16 for s, x in zip(t.stride()[:-1], t.shape[:-1]) if x > 1):
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Element strides of all but the last dimension; a dimension of one element does not step."""
    return tuple(s if x > 1 else 0 for s, x in zip(t.stride()[:-1], t.shape[:-1]))


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def _check_slopes(slopes: Optional[torch.Tensor], h_q: int) -> Optional[torch.Tensor]:
    if slopes is None:
        return None
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (h_q,):
        raise ValueError(f"slopes must be float32 [{h_q}]")
    if slopes.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("slopes get no gradient: detach them")
    return slopes.contiguous()


def mask_spans(n: int, batch: int, n_q: int, q_pos0: int, causal: bool, doc_starts: Optional[torch.Tensor],
               prefix_lens: Optional[torch.Tensor], device: torch.device) -> torch.Tensor:
    """Key interval of each row, int32 [batch, n_q, 2] (ssa_mask_spans)."""
    out = torch.empty((batch, n_q, 2), device=device, dtype=torch.int32)
    _same_device(spans=out, doc_starts=doc_starts, prefix_lens=prefix_lens)
    docs = 1 if doc_starts is None else doc_starts.shape[-1] - 1
    if doc_starts is not None:
        if doc_starts.dim() != 2 or doc_starts.shape[0] != batch or docs < 1:
            raise ValueError(f"doc_starts must be [{batch}, documents + 1], got {tuple(doc_starts.shape)}")
        doc_starts = _index32(doc_starts, "doc_starts")
    if prefix_lens is not None:
        if tuple(prefix_lens.shape) != (batch, docs):
            raise ValueError(f"prefix_lens must be [{batch}, {docs}], got {tuple(prefix_lens.shape)}")
        prefix_lens = _index32(prefix_lens, "prefix_lens")
    _call_on(out, "ssa_mask_spans", ptr(doc_starts), docs, ptr(prefix_lens), batch, n, n_q, q_pos0, int(bool(causal)),
             ptr(out), stream_of(out))
    return out


def _index32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    return t.to(torch.int32).contiguous()


def _check_dense(q, k, v, spans) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [B, n, heads, d], got shape {tuple(t.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    B, n_q, h_q, d = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != d:
        raise ValueError(f"k and v must be [{B}, n, h_kv, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[2] == 0 or h_q % k.shape[2] != 0:
        raise ValueError(f"{h_q} query heads are not divisible by {k.shape[2]} KV heads")
    if spans is not None and (spans.dtype != torch.int32 or tuple(spans.shape) != (B, n_q, 2) or not spans.is_contiguous()):
        raise ValueError(f"spans must be a contiguous int32 [{B}, {n_q}, 2] tensor")


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, spans: Optional[torch.Tensor] = None,
                     scale_div: Optional[float] = None, softcap: float = 0.0,
                     slopes: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None, with_lse: bool = False):
    """Dense attention over each row's key interval (ssa_masked_attention): [B, n_q, h_q, d]
    in q's dtype.  ``with_lse`` returns (out, out_low, lse) for the backward: what rounding left of a
    bf16 output (None for float32) and the float32 [B, h_q, n_q] log2 sums.
    ``spans`` None: causal.  Query row i sits at key position ``q_pos0 + i`` (default n - n_q)."""
    _same_device(q=q, k=k, v=v, spans=spans, slopes=slopes)
    _check_dense(q, k, v, spans)
    B, n_q, h_q, d = q.shape
    n, h_kv = k.shape[1], k.shape[2]
    slopes = _check_slopes(slopes, h_q)
    if q_pos0 is None:
        q_pos0 = n - n_q
    q, k, v = _aligned_rows(q), _aligned_rows(k), _aligned_rows(v)
    out = torch.empty((B, n_q, h_q, d), device=q.device, dtype=q.dtype)
    lse = torch.empty((B, h_q, n_q), device=q.device, dtype=torch.float32) if with_lse else None
    low = torch.empty_like(out) if with_lse and q.dtype == torch.bfloat16 else None
    nbytes = int(_lib.load().ssa_masked_attention_workspace_bytes(_lib.elem_dtype(q), B, n, n_q, h_q, h_kv, d))
    ws = _workspace(nbytes, q.device)
    _call_on(q, "ssa_masked_attention", ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), B, n, n_q, q_pos0, h_q, h_kv, d,
             *_strides(q), *_strides(k), *_strides(v), ptr(spans), float(math.sqrt(d) if scale_div is None else scale_div),
             float(softcap), ptr(slopes), ptr(out), *_strides(out), ptr(low), ptr(lse), ptr(ws), nbytes, stream_of(q))
    return (out, low, lse) if with_lse else out


def masked_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, dout: torch.Tensor,
                              lse: torch.Tensor, spans: Optional[torch.Tensor] = None, scale_div: Optional[float] = None,
                              softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, q_pos0: Optional[int] = None,
                              out_low: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of masked_attention w.r.t. q, k and v, in their dtype and contiguous, from the
    forward's ``out``, ``lse`` and (bf16) ``out_low`` and the output gradient."""
    _same_device(q=q, k=k, v=v, out=out, dout=dout, lse=lse, spans=spans, slopes=slopes, out_low=out_low)
    _check_dense(q, k, v, spans)
    B, n_q, h_q, d = q.shape
    n, h_kv = k.shape[1], k.shape[2]
    if tuple(out.shape) != (B, n_q, h_q, d) or tuple(dout.shape) != (B, n_q, h_q, d):
        raise ValueError("out and dout must have q's shape")
    if out.dtype != q.dtype or dout.dtype != q.dtype:
        raise TypeError(f"out and dout must have q's dtype {q.dtype}")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, h_q, n_q) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 [{B}, {h_q}, {n_q}] tensor")
    slopes = _check_slopes(slopes, h_q)
    if q_pos0 is None:
        q_pos0 = n - n_q
    dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    if out_low is not None and (out_low.shape != out.shape or out_low.dtype != out.dtype or out_low.stride() != out.stride()):
        raise ValueError("out_low must have out's shape, strides and dtype")
    q, k, v, out, dout = (_aligned_rows(t) for t in (q, k, v, out, dout))
    out_low = None if out_low is None else _aligned_rows(out_low)
    nbytes = int(_lib.load().ssa_masked_attention_backward_workspace_bytes(_lib.elem_dtype(q), B, n, n_q, h_q, h_kv, d))
    ws = _workspace(nbytes, q.device)
    _call_on(q, "ssa_masked_attention_backward", ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), B, n, n_q, q_pos0, h_q, h_kv,
             d, *_strides(q), *_strides(k), *_strides(v), ptr(spans),
             float(math.sqrt(d) if scale_div is None else scale_div), float(softcap), ptr(slopes), ptr(out), ptr(out_low),
             *_strides(out), ptr(dout), *_strides(dout), ptr(lse), ptr(dq), ptr(dk), ptr(dv), ptr(ws), nbytes, stream_of(q))
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
    _same_device(q=q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, table=table, starts=starts, cached=cached, slopes=slopes,
                 out=out, error_flag=error_flag)
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("q must be [T, h_q, d] and the pools [pages, page size, h_kv, d]")
    T, h_q, d = q.shape
    pages, page, h_kv, _ = k_pages.shape
    if k_pages.shape[3] != d or h_kv == 0 or h_q % h_kv != 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit pages {tuple(k_pages.shape)}")
    for name, t in (("k", k), ("v", v)):
        if t is not None and tuple(t.shape) != (T, h_kv, d):
            raise ValueError(f"{name} must be [{T}, {h_kv}, {d}], got {tuple(t.shape)}")
    for name, t in (("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("out", out)):
        if t is not None and t.dtype != q.dtype:
            raise TypeError(f"{name} must have q's dtype {q.dtype}, got {t.dtype}")
    B = table.shape[0]
    for name, t, shape in (("table", table, (B, table.shape[-1])), ("starts", starts, (B + 1,)), ("cached", cached, (B,))):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or (t.shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name} must be an int32 {list(shape)} tensor with contiguous rows")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        e = t.element_size()
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * e % 16 for s in _strides(t)):
            raise ValueError(f"{name} must have contiguous rows aligned to 16 bytes")
    slopes = _check_slopes(slopes, h_q)
    if error_flag is not None and (error_flag.dtype != torch.int32 or error_flag.numel() != 1):
        raise ValueError("error_flag must be one int32")
    q = _aligned_rows(q)
    k, v = (t if t is None else _aligned_rows(t) for t in (k, v))
    if out is None:
        out = torch.empty((T, h_q, d), device=q.device, dtype=q.dtype)
    elif tuple(out.shape) != (T, h_q, d) or _aligned_rows(out) is not out:
        raise ValueError(f"out must be [{T}, {h_q}, {d}] with rows aligned to 16 bytes")
    max_new = T if max_new is None else min(int(max_new), T)
    width = table.shape[1] * page
    max_len = width if max_len is None else min(int(max_len), width)
    nbytes = int(_lib.load().ssa_paged_step_workspace_bytes(_lib.elem_dtype(q), T, B, h_q, h_kv, d, max_new, max_len))
    ws = _workspace(nbytes, q.device)
    ks, vs = ((0, 0) if t is None else _strides(t) for t in (k, v))
    _call_on(q, "ssa_paged_step", ptr(q), ptr(k), ptr(v), _lib.elem_dtype(q), T, B, h_q, h_kv, d, *_strides(q), *ks, *vs,
             ptr(k_pages), ptr(v_pages), pages, page, *_strides(k_pages), *_strides(v_pages), ptr(table),
             table.stride(0) if B > 1 else 0, table.shape[1], ptr(starts), ptr(cached), max_new, max_len,
             float(math.sqrt(d) if scale_div is None else scale_div), float(softcap), ptr(slopes), ptr(out), *_strides(out),
             ptr(error_flag), ptr(ws), nbytes, stream_of(q))
    return out


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, sections,
              inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions with several axes on q [B, n, h_q, d] and k [B, n, h_k, d] (or None)
    (ssa_rope_axes): positions int [axes, B, n], freqs float64 [rot / 2], sections the pairs
    of each axis.  New contiguous tensors of q's dtype; ``inverse`` applies the transpose."""
    _same_device(q=q, k=k, positions=positions, freqs=freqs)
    for name, t in (("q", q), ("k", k)):
        if t is not None and t.dim() != 4:
            raise ValueError(f"{name} must be [B, n, heads, d], got shape {tuple(t.shape)}")
    B, n, h_q, d = q.shape
    if k is not None and (k.shape[:2] != q.shape[:2] or k.shape[3] != d or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    axes = len(sections)
    if tuple(positions.shape) != (axes, B, n):
        raise ValueError(f"positions must be [{axes}, {B}, {n}], got {tuple(positions.shape)}")
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("freqs must be float64 [rot / 2] (axis_rope_freqs)")
    pos_dtype = _lib.index_dtype(positions)
    if n > 1 and positions.stride(2) != 1:
        positions = positions.contiguous()
    freqs = freqs.contiguous()
    q, k = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    qo = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    ko = None if k is None else torch.empty(k.shape, device=q.device, dtype=q.dtype)
    cuts = (ctypes.c_int32 * axes)(*(int(x) for x in sections))
    none = (0, 0, 0)
    _call_on(q, "ssa_rope_axes", ptr(q), ptr(k), _lib.elem_dtype(q), B, n, h_q, 0 if k is None else k.shape[2], d,
             *_strides(q), *(none if k is None else _strides(k)), ptr(positions), pos_dtype, *_strides(positions), axes,
             cuts, ptr(freqs), 2 * freqs.shape[0], int(bool(inverse)), ptr(qo), *_strides(qo), ptr(ko),
             *(none if ko is None else _strides(ko)), stream_of(q))
    return qo, ko
