"""A paged K/V cache and the attention of new tokens over it.

``SSADecodeCache`` holds one contiguous buffer per batch element and selects keys; the
dense layers beside it, and batches whose sequences come and go, keep their keys in
pages of a shared pool.  ``paged_step`` is one call for a ragged batch (chunks of
prompts and single tokens together); ``PagedKVCache`` keeps the pool, the tables and
the lengths.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib, kernels


def paged_step(q: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor], k_pages: torch.Tensor,
               v_pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, cached: torch.Tensor, *,
               scale: Optional[float] = None, softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
               max_new: Optional[int] = None, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
               check: bool = False) -> torch.Tensor:
    """Append a ragged batch's new tokens to their pages and attend them; ``[T, h_q, d]``.

    Sequence b's new tokens are rows ``starts[b]`` to ``starts[b + 1]`` of ``q [T, h_q, d]``
    and ``k, v [T, h_kv, d]``; its key j is row ``j % page_size`` of page ``table[b, j //
    page_size]`` of ``k_pages, v_pages [pages, page_size, h_kv, d]`` (strided pools too), and
    it has ``cached[b]`` keys already.  k and v are written behind them (pass None where they
    are there already), and each new token attends every key up to its own, with
    ``masked_attention``'s scores (``scale``, ``softcap``, ``slopes``).

    ``table`` [B, width], ``starts`` [B + 1] and ``cached`` [B] are int32 on the device and
    read by the kernels, so a captured call follows them.  ``max_new`` and ``max_len`` say how
    many new tokens and keys (the new ones included) a sequence has at most: the work is laid
    out for them (defaults: T, and what the table holds).  A sequence that breaks a bound is
    left out; ``check=True`` waits for the device and raises IndexError then, or if a page lies
    outside the pool.  Rows of no sequence, and of one that is left out, keep what ``out`` held,
    and are zeros where it was not given.

    float32 and bfloat16 (pools of the same dtype), head_dim a multiple of 8 up to 128,
    page_size a power of 2 from 8 to 4096.  No gradient: inputs that want one are refused (call
    it under ``torch.no_grad()``, or detach them)."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or
                                    any([t.requires_grad for t in (k, v, slopes, out) if t is not None])):
        raise NotImplementedError("paged_step has no gradient: call it under torch.no_grad(), or detach its inputs")
    _lib.refuse_tangents("paged_step", q, k, v, k_pages, v_pages, slopes)
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    flag = torch.zeros(1, device=q.device, dtype=torch.int32) if check else None
    out = kernels.paged_step(q, k, v, k_pages, v_pages, table, starts, cached, scale, softcap or 0.0, slopes, max_new,
                             max_len, out, flag)
    if flag is not None and int(flag.item()) != 0:
        raise IndexError("paged_step: a sequence exceeds its bounds or a page lies outside the pool")
    return out


class PagedKVCache:
    """Pages of K and V for sequences that come and go.

    ``add()`` opens a sequence, ``step`` appends and attends tokens of any of them,
    ``free`` gives its pages back.  The tables are kept on the host: ``step`` copies them to
    the device and waits for the stream to do so (about half a millisecond of the host's for 32
    sequences of 8191 keys), once a layer, and cannot be captured.  A program that calls
    several layers with one set of tables, or captures its steps, keeps them on the device
    and calls ``paged_step``.  288 GB of HBM hold, at h_kv = 8, d = 128 in bf16, the
    pages of about 70 M tokens of one layer."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        if page_size < 8 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of 2 in [8, 4096], got {page_size}")
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {head_dim}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        device = torch.device("cuda" if device is None else device)
        self.page_size = page_size
        self.k_pages = torch.empty(num_pages, page_size, num_kv_heads, head_dim, device=device, dtype=dtype)
        self.v_pages = torch.empty_like(self.k_pages)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}   # sequence -> its pages, in order
        self._len = {}     # sequence -> its keys
        self._next = 0

    def add(self) -> int:
        """Opens a sequence and returns its number."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        """Closes a sequence; its pages are used again."""
        del self._len[seq]
        self._free.extend(reversed(self._pages.pop(seq)))

    def length(self, seq: int) -> int:
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqs: Sequence[int], counts: Sequence[int],
             *, scale: Optional[float] = None, softcap: Optional[float] = None,
             slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Appends ``counts[i]`` tokens to sequence ``seqs[i]``, in order the rows of
        ``q [T, h_q, d]``, ``k, v [T, h_kv, d]``, and returns their attention ``[T, h_q, d]``
        over everything their sequences hold.  Raises ValueError, with nothing changed, when
        the pool has too few pages left."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("seqs and counts must pair distinct sequences with token counts")
        if sum(counts) != q.shape[0]:
            raise ValueError(f"counts add up to {sum(counts)} tokens, q holds {q.shape[0]}")
        if any(s not in self._len for s in seqs):
            raise ValueError("a sequence is not open")
        if not seqs or q.shape[0] == 0:
            return q.new_empty(q.shape)
        P = self.page_size
        need = [-(-(self._len[s] + c) // P) - len(self._pages[s]) for s, c in zip(seqs, counts)]
        if sum(x for x in need if x > 0) > len(self._free):
            raise ValueError(f"cache full: {sum(x for x in need if x > 0)} pages needed, {len(self._free)} free")
        before = {s: len(self._pages[s]) for s in seqs}
        for s, x in zip(seqs, need):
            for _ in range(x):
                self._pages[s].append(self._free.pop())
        try:
            B, width = len(seqs), max(1, max(len(self._pages[s]) for s in seqs))
            host = torch.zeros(2 * B + 1 + B * width, dtype=torch.int32)
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c)
            host[:B + 1] = torch.tensor(starts, dtype=torch.int32)
            host[B + 1:2 * B + 1] = torch.tensor([self._len[s] for s in seqs], dtype=torch.int32)
            rows = host[2 * B + 1:].view(B, width)
            for i, s in enumerate(seqs):
                rows[i, :len(self._pages[s])] = torch.tensor(self._pages[s], dtype=torch.int32)
            dev = host.to(self.k_pages.device)
            out = paged_step(q, k, v, self.k_pages, self.v_pages, dev[2 * B + 1:].view(B, width), dev[:B + 1],
                             dev[B + 1:2 * B + 1], scale=scale, softcap=softcap, slopes=slopes, max_new=max(counts),
                             max_len=max(self._len[s] + c for s, c in zip(seqs, counts)))
        except Exception:
            for s in seqs:  # nothing was appended: the new pages go back
                while len(self._pages[s]) > before[s]:
                    self._free.append(self._pages[s].pop())
            raise
        for s, c in zip(seqs, counts):
            self._len[s] += c
        return out
