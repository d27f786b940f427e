"""A paged K/V cache and the attention of new tokens over it.

``SSADecodeCache`` holds one contiguous buffer per batch element and selects keys; the
dense layers beside it, and batches whose sequences come and go, keep their keys in
pages of a shared pool.  ``paged_step`` is one call for a ragged batch (chunks of
prompts and single tokens together); ``PagedKVCache`` keeps the pool, the tables and
the lengths.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib, kernels


def paged_step(q: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor], k_pages: torch.Tensor,
               v_pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, cached: torch.Tensor, *,
               scale: Optional[float] = None, softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
               max_new: Optional[int] = None, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
               check: bool = False, window: Optional[int] = None, sinks: int = 0,
               parents: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None,
               v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
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

    ``window`` w limits a token at position p to the keys at positions p - w + 1 to p and the
    first ``sinks`` positions (up to its own); pages that hold none of these are not read, and
    their table entries may hold anything.

    ``parents`` (int32 [T] on the device) makes a sequence's new tokens drafts in a tree: its
    i-th one follows its new token ``parents[starts[b] + i]`` < i, or the cached ones where that
    is -1.  It attends the cached keys, its ancestors and itself, from position ``cached[b]`` +
    the number of its ancestors; its key is written to ``cached[b] + i`` as ever, and
    ``paged_keep`` then puts the path that is kept in order.  At most 64 drafts a sequence
    (``max_new``'s default then).  A parent that does not come before its token counts as -1, and
    as a broken bound for ``check``.

    Pools of int8 or float8_e4m3fn hold codes, with ``k_scales, v_scales`` float32 [pages,
    page_size, h_kv] (any strides): a row stands for code * scale, and is written with scale =
    max |x| / 127 (or / 448) and the nearest codes.  New tokens are attended as they are given and
    held in 8 bits from then on.  Rows below 2^-100 are held as zeros, and a row with an infinity or NaN as NaN.

    float32 and bfloat16 (other pools of the same dtype), head_dim a multiple of 8 up to 128,
    page_size a power of 2 from 8 to 4096.  No gradient: inputs that want one are refused (call
    it under ``torch.no_grad()``, or detach them)."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or
                                    (k is not None and (k.requires_grad or v is not None and v.requires_grad)) or
                                    any([t.requires_grad for t in (slopes, out, k_scales, v_scales) if t is not None])):
        raise NotImplementedError("paged_step has no gradient: call it under torch.no_grad(), or detach its inputs")
    _lib.refuse_tangents("paged_step", q, k, v, k_pages, v_pages, slopes, k_scales, v_scales, out)
    window, sinks = (0, 0) if window is None and sinks == 0 else (_window(window, sinks), min(int(sinks), 1 << 31))
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    flag = torch.zeros(1, device=q.device, dtype=torch.int32) if check else None
    out = kernels.paged_step(q, k, v, k_pages, v_pages, table, starts, cached, scale, softcap or 0.0, slopes, max_new,
                             max_len, out, flag, window, sinks, parents, k_scales, v_scales)
    if flag is not None and int(flag.item()) != 0:
        raise IndexError("paged_step: a sequence exceeds its bounds or a page lies outside the pool")
    return out


def _window(window: Optional[int], sinks: int) -> int:
    """The window as the kernels take it (0: none)."""
    if window is not None and window < 1:
        raise ValueError(f"window must be positive, got {window}")
    if sinks < 0 or (sinks > 0 and window is None):
        raise ValueError(f"sinks must not be negative and go with a window, got sinks={sinks}, window={window}")
    return 0 if window is None else min(int(window), 1 << 31)


def paged_read(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, first: torch.Tensor,
               tokens: int, *, dtype: Optional[torch.dtype] = None, k_scales: Optional[torch.Tensor] = None,
               v_scales: Optional[torch.Tensor] = None, check: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of a paged cache read back: ``(k, v)``, each ``[tokens, h_kv, d]``.

    Row ``starts[b] + i`` is key ``first[b] + i`` of sequence b, up to row ``starts[b + 1]``; rows of
    no sequence are zeros.  ``table``, ``starts`` [B + 1] and ``first`` [B] are int32 on the device.
    Pools of 8 bits (with their scales) are read as ``dtype`` (bfloat16, or float32), rounded once,
    others as they are.  A key past the table or in a page outside the pool is zeros;
    ``check=True`` waits for the device and raises IndexError then.  No gradient."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (k_pages, v_pages, k_scales, v_scales)):
        raise NotImplementedError("paged_read has no gradient: call it under torch.no_grad(), or detach its inputs")
    _lib.refuse_tangents("paged_read", k_pages, v_pages, k_scales, v_scales)
    flag = torch.zeros(1, device=k_pages.device, dtype=torch.int32) if check else None
    res = kernels.paged_read(k_pages, v_pages, table, starts, first, int(tokens), dtype, k_scales, v_scales, flag)
    if flag is not None and int(flag.item()) != 0:
        raise IndexError("paged_read: a key lies past its table or outside the pool")
    return res


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, cached: torch.Tensor, kept: torch.Tensor, *,
               k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None, check: bool = False) -> None:
    """Keeps some of the tokens that a ``paged_step`` with ``parents`` wrote, in place.

    ``kept`` (int32 [B, most kept] on the device, at most 64) names the new tokens of each sequence
    that stay, ascending, up to the first -1: the accepted path from a root on.  Key ``cached[b] +
    kept[b, t]`` goes to key ``cached[b] + t``, and the sequence then has ``cached[b]`` + as many
    keys.  An entry that does not ascend ends its sequence's; ``check=True`` waits for the device
    and raises IndexError then, or if a key lies past the table or outside the pool."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (k_pages, v_pages, k_scales, v_scales)):
        raise NotImplementedError("paged_keep has no gradient: call it under torch.no_grad(), or detach its inputs")
    _lib.refuse_tangents("paged_keep", k_pages, v_pages, k_scales, v_scales)
    flag = torch.zeros(1, device=k_pages.device, dtype=torch.int32) if check else None
    kernels.paged_keep(k_pages, v_pages, table, cached, kept, k_scales, v_scales, flag)
    if flag is not None and int(flag.item()) != 0:
        raise IndexError("paged_keep: kept does not ascend, or a key lies past its table or outside the pool")


class PagedKVCache:
    """Pages of K and V for sequences that come and go.

    ``add()`` opens a sequence, ``step`` appends and attends tokens of any of them,
    ``free`` gives its pages back.  The tables are kept on the host: ``step`` copies them to
    the device and waits for the stream to do so (about half a millisecond of the host's for 32
    sequences of 8191 keys), once a layer, and cannot be captured.  A program that calls
    several layers with one set of tables, or captures its steps, keeps them on the device
    and calls ``paged_step``.  288 GB of HBM hold, at h_kv = 8, d = 128 in bf16, the
    pages of about 70 M tokens of one layer.

    ``dtype`` int8 or float8_e4m3fn holds the rows in 8 bits with a scale each (135 M tokens).
    With ``window`` (and ``sinks``) every step attends as ``paged_step`` does with them, and a
    sequence's pages that no later token sees go back to the pool as it grows (its table keeps their
    entries, 4 bytes a page that are copied with a step).  ``step`` with
    ``parents`` verifies drafted trees, and ``keep`` then says what stays of them."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None, *, window: Optional[int] = None, sinks: int = 0):
        if page_size < 8 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of 2 in [8, 4096], got {page_size}")
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {head_dim}")
        if dtype not in (torch.float32, torch.bfloat16, *kernels.HELD_DTYPES):
            raise TypeError(f"dtype must be float32 or bfloat16, or int8 or float8_e4m3fn, got {dtype}")
        _window(window, sinks)
        device = torch.device("cuda" if device is None else device)
        self.page_size, self.window, self.sinks = page_size, window, sinks
        self.k_pages = torch.empty(num_pages, page_size, num_kv_heads, head_dim, device=device, dtype=dtype)
        self.v_pages = torch.empty_like(self.k_pages)
        self.k_scales = self.v_scales = None
        if dtype in kernels.HELD_DTYPES:  # a head's scales of a page's tokens are neighbours
            self.k_scales, self.v_scales = (torch.empty(num_pages, num_kv_heads, page_size, device=device).transpose(1, 2)
                                            for _ in "kv")
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}   # sequence -> its pages, in order (0 where one was given back)
        self._gone = {}    # sequence -> which of them were
        self._len = {}     # sequence -> its keys
        self._drafts = {}  # sequence -> drafted tokens at its end, of which keep says what stays
        self._parents = {}  # sequence -> those tokens' parents
        self._next = 0

    def add(self) -> int:
        """Opens a sequence and returns its number."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._gone[seq], self._len[seq], self._drafts[seq] = [], set(), 0, 0
        return seq

    def free(self, seq: int) -> None:
        """Closes a sequence; its pages are used again."""
        del self._len[seq], self._drafts[seq]
        self._parents.pop(seq, None)
        gone = self._gone.pop(seq)
        self._free.extend(reversed([x for i, x in enumerate(self._pages.pop(seq)) if i not in gone]))

    def length(self, seq: int) -> int:
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _behind(self, seq: int) -> list:
        """Pages of a sequence that neither its next token nor a later one sees."""
        if self.window is None:
            return []
        P = self.page_size
        first, last = -(-self.sinks // P), (self._len[seq] + 1 - self.window) // P  # (whole pages before the window)
        at = end = min(last, len(self._pages[seq]))
        while at > first and at - 1 not in self._gone[seq]:  # (those given back are the ones from `first` on)
            at -= 1
        return list(range(at, end))

    def _tables(self, seqs: Sequence[int], *rows: Sequence[int]):
        """The sequences' table [B, width] and the given rows of numbers, on the device by one copy."""
        B, width = len(seqs), max(1, max(len(self._pages[s]) for s in seqs))
        sizes = [len(r) for r in rows]
        host = torch.zeros(sum(sizes) + B * width, dtype=torch.int32)
        at = 0
        for r in rows:
            host[at:at + len(r)] = torch.tensor(r, dtype=torch.int32)
            at += len(r)
        table = host[at:].view(B, width)
        for i, s in enumerate(seqs):
            pages, gone = self._pages[s], len(self._gone[s])
            first = -(-self.sinks // self.page_size) if gone else len(pages)
            table[i, :first] = torch.tensor(pages[:first], dtype=torch.int32)
            if gone:  # (entries of pages that were given back stay 0: only live ones are walked)
                table[i, first + gone:len(pages)] = torch.tensor(pages[first + gone:], dtype=torch.int32)
        dev = host.to(self.k_pages.device)
        return dev[at:].view(B, width), *dev[:at].split(sizes)

    def _scales(self) -> dict:
        return {} if self.k_scales is None else {"k_scales": self.k_scales, "v_scales": self.v_scales}

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqs: Sequence[int], counts: Sequence[int],
             *, scale: Optional[float] = None, softcap: Optional[float] = None,
             slopes: Optional[torch.Tensor] = None, parents: Optional[Sequence[Sequence[int]]] = None) -> torch.Tensor:
        """Appends ``counts[i]`` tokens to sequence ``seqs[i]``, in order the rows of
        ``q [T, h_q, d]``, ``k, v [T, h_kv, d]``, and returns their attention ``[T, h_q, d]``
        over everything their sequences hold (their window's).  ``parents`` (for each sequence its
        tokens' parents, -1: the cached ones) makes them drafts: ``keep`` has to follow before the
        sequence's next step.  Raises ValueError, with nothing changed, when the pool has too few
        pages left."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("seqs and counts must pair distinct sequences with token counts")
        if sum(counts) != q.shape[0]:
            raise ValueError(f"counts add up to {sum(counts)} tokens, q holds {q.shape[0]}")
        if any(s not in self._len for s in seqs):
            raise ValueError("a sequence is not open")
        if any(self._drafts[s] for s in seqs):
            raise ValueError("a sequence has drafted tokens: keep says which of them stay")
        if parents is not None:
            if [len(x) for x in parents] != list(counts) or any(not -1 <= y < i for x in parents for i, y in enumerate(x)):
                raise ValueError("parents must name, for every token of each sequence, -1 or a token before it")
            if any(c > 64 for c in counts):
                raise ValueError("a sequence takes at most 64 drafted tokens")
        if not seqs or q.shape[0] == 0:
            return q.new_empty(q.shape)
        P = self.page_size
        behind = {s: self._behind(s) for s in seqs}
        need = [max(0, -(-(self._len[s] + c) // P) - len(self._pages[s])) for s, c in zip(seqs, counts)]
        have = len(self._free) + sum(len(x) for x in behind.values())
        if sum(need) > have:
            raise ValueError(f"cache full: {sum(need)} pages needed, {have} free")
        before = {s: len(self._pages[s]) for s in seqs}
        for s in seqs:  # (the kernels do not read them: another sequence may write to them in this call)
            for i in behind[s]:
                self._free.append(self._pages[s][i])
                self._pages[s][i] = 0
                self._gone[s].add(i)
        for s, x in zip(seqs, need):
            for _ in range(x):
                self._pages[s].append(self._free.pop())
        try:
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c)
            drafts = [] if parents is None else [y for x in parents for y in x]
            table, starts, cached, drafts = self._tables(seqs, starts, [self._len[s] for s in seqs], drafts)
            out = paged_step(q, k, v, self.k_pages, self.v_pages, table, starts, cached, scale=scale, softcap=softcap,
                             slopes=slopes, max_new=max(counts),
                             max_len=max(self._len[s] + c for s, c in zip(seqs, counts)), window=self.window,
                             sinks=self.sinks, parents=None if parents is None else drafts, **self._scales())
        except Exception:
            for s in seqs:  # nothing was appended: the new pages go back
                while len(self._pages[s]) > before[s]:
                    self._free.append(self._pages[s].pop())
            raise
        for i, (s, c) in enumerate(zip(seqs, counts)):
            self._len[s] += c
            if parents is not None:
                self._drafts[s], self._parents[s] = c, list(parents[i])
        return out

    def keep(self, seqs: Sequence[int], kept: Sequence[Sequence[int]]) -> None:
        """Says which of the tokens that the last ``step`` of each sequence drafted stay: ``kept[i]``
        are their numbers, ascending, a path from a root of the tree on (empty: none).  The rest is
        dropped, and pages it had filled go back.  Raises ValueError, with nothing changed, for
        tokens that are no such path: each but the first follows the one before it."""
        if len(seqs) != len(kept) or len(set(seqs)) != len(seqs) or any(s not in self._len for s in seqs):
            raise ValueError("seqs and kept must pair distinct open sequences with tokens")
        for s, x in zip(seqs, kept):
            if any(not a < b for a, b in zip([-1, *x], [*x, self._drafts[s]])):
                raise ValueError(f"kept tokens must ascend and lie among the {self._drafts[s]} drafted ones")
            up = self._parents.get(s)
            if up is not None and any(up[b] != a for a, b in zip([-1, *x], x)):
                raise ValueError(f"kept tokens must be a path from a root of the tree on, not {list(x)} of parents {up}")
        if not seqs:
            return
        base = {s: self._len[s] - self._drafts[s] for s in seqs}
        if any(list(x) != list(range(len(x))) for x in kept):
            most = max(len(x) for x in kept)
            flat = [y for x in kept for y in [*x, *[-1] * (most - len(x))]]
            table, cached, rows = self._tables(seqs, [base[s] for s in seqs], flat)
            paged_keep(self.k_pages, self.v_pages, table, cached, rows.view(len(seqs), most), **self._scales())
        for s, x in zip(seqs, kept):
            self._len[s], self._drafts[s] = base[s] + len(x), 0
            self._parents.pop(s, None)
            while len(self._pages[s]) > -(-self._len[s] // self.page_size):
                self._free.append(self._pages[s].pop())

    def read(self, seq: int, first: int = 0, last: Optional[int] = None, *, dtype: Optional[torch.dtype] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys ``first`` to ``last`` (default: all) of a sequence as the cache holds them, ``(k, v)`` each
        ``[last - first, h_kv, d]``; pages of 8 bits as ``dtype`` (bfloat16, or float32)."""
        last = self._len[seq] if last is None else last
        if not 0 <= first <= last <= self._len[seq]:
            raise ValueError(f"keys {first} to {last} of a sequence of {self._len[seq]}")
        P = self.page_size
        if any(first < (i + 1) * P and i * P < last for i in self._gone[seq]):
            raise ValueError("some of these keys were given back: no token sees them any more")
        if first == last:
            _, _, h_kv, d = self.k_pages.shape
            dtype = dtype or (torch.bfloat16 if self.k_scales is not None else self.k_pages.dtype)
            return tuple(self.k_pages.new_empty((0, h_kv, d), dtype=dtype) for _ in "kv")
        table, starts, at = self._tables([seq], [0, last - first], [first])
        return paged_read(self.k_pages, self.v_pages, table, starts, at, last - first, dtype=dtype, **self._scales())
