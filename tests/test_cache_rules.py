"""Rules of the paged cache's calls that need no kernel: what they refuse, and the books of PagedKVCache."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import ssa_amd


def test_step_refuses_every_tangent_that_it_would_drop():
    z = torch.zeros
    q, k = z(3, 4, 64), z(3, 2, 64)
    codes, scales = z(5, 16, 2, 64, dtype=torch.int8), z(5, 16, 2)
    table, starts, cached = z(1, 5, dtype=torch.int32), z(2, dtype=torch.int32), z(1, dtype=torch.int32)
    floats = dict(q=q, k=k, v=k.clone(), slopes=z(4), k_scales=scales, v_scales=scales.clone(), out=z(3, 4, 64))
    rest = dict(k_pages=codes, v_pages=codes.clone(), table=table, starts=starts, cached=cached)
    with fwAD.dual_level():
        for name, t in floats.items():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ssa_amd.paged_step(**{**floats, **rest, name: fwAD.make_dual(t, torch.ones_like(t))})
        with pytest.raises(RuntimeError, match="GPU"):  # (no tangent: the device is what is wrong)
            ssa_amd.paged_step(**floats, **rest)


def _drafted(monkeypatch, parents, dtype=torch.bfloat16):
    """A cache on the host after a step that drafted trees of these parents (no kernel runs)."""
    moved = []
    monkeypatch.setattr(ssa_amd.paged, "paged_step", lambda q, *a, **kw: torch.zeros_like(q))
    monkeypatch.setattr(ssa_amd.paged, "paged_keep", lambda *a, **kw: moved.append(a))
    c = ssa_amd.PagedKVCache(20, 16, 2, 64, dtype=dtype, device="cpu")
    seqs = [c.add() for _ in parents]
    for s in seqs:
        x = torch.zeros(5, 2, 64, dtype=dtype)
        c.step(torch.zeros(5, 4, 64, dtype=dtype), x, x, [s], [5])
    T = sum(len(p) for p in parents)
    x = torch.zeros(T, 2, 64, dtype=dtype)
    c.step(torch.zeros(T, 4, 64, dtype=dtype), x, x, seqs, [len(p) for p in parents], parents=parents)
    return c, seqs, moved


def test_keep_takes_a_path_of_the_tree_alone(monkeypatch):
    tree = [-1, 0, 0, 1, -1, 4, 3]
    for bad in ([0, 1, 2], [1], [0, 3], [0, 4], [4, 6], [0, 1, 3, 5], [2, 6]):
        c, (a, b), moved = _drafted(monkeypatch, [tree, [-1, 0]])
        books = (c.length(a), c.length(b), c.free_pages)
        with pytest.raises(ValueError, match="path"):
            c.keep([b, a], [[0], bad])
        assert not moved and books == (c.length(a), c.length(b), c.free_pages)
        c.keep([a, b], [[], [0, 1]])  # (and may still say what stays)
        assert (c.length(a), c.length(b)) == (5, 7)
    for good in ([], [0], [4], [0, 2], [4, 5], [0, 1, 3, 6]):
        c, (a, b), moved = _drafted(monkeypatch, [tree, [-1, 0]])
        c.keep([a, b], [good, [0, 1]])
        assert c.length(a) == 5 + len(good) and len(moved) == (0 if good in ([], [0]) else 1)
        # the next step drafts another tree, of which another path stays
        x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
        c.step(torch.zeros(3, 4, 64, dtype=torch.bfloat16), x, x, [a], [3], parents=[[-1, -1, 1]])
        with pytest.raises(ValueError, match="path"):
            c.keep([a], [[0, 1]])
        c.keep([a], [[1, 2]])
        assert c.length(a) == 7 + len(good)
        c.free(a)
        assert a not in c._parents


class _Counted(set):
    asked = 0

    def __contains__(self, x):
        type(self).asked += 1
        return super().__contains__(x)


@pytest.mark.parametrize("window,sinks", [(40, 17), (1, 0), (100, 16), (33, 1)])
def test_a_step_behind_a_window_walks_live_pages_alone(monkeypatch, window, sinks):
    """The host's work of a step does not grow with the pages that its sequence has left behind, and the table
    that it makes has every page that some token sees."""
    tables = []
    monkeypatch.setattr(ssa_amd.paged, "paged_step", lambda q, k, v, kp, vp, table, *a, **kw: (tables.append(table.clone()), torch.zeros_like(q))[1])
    c = ssa_amd.PagedKVCache(40, 16, 2, 64, device="cpu", window=window, sinks=sinks)
    s, other = c.add(), c.add()
    c._gone[s] = _Counted()
    q, k = torch.zeros(17, 4, 64), torch.zeros(17, 2, 64)
    length, given = 0, set()
    for step in range(400):
        m = (1, 17, 5)[step % 3]
        _Counted.asked = 0
        c.step(q[:m], k[:m], k[:m], [other, s], [0, m])
        assert _Counted.asked <= 4, "pages behind the window are asked for again"
        pages, table = c._pages[s], tables.pop()
        live = {j // 16 for j in range(length, length + m)}  # (new keys are written)
        for p in range(length, length + m):
            live |= {j // 16 for j in range(max(0, p + 1 - window), p + 1)} | {j // 16 for j in range(min(sinks, p + 1))}
        given |= {i for i in range(len(pages)) if i in set(c._gone[s])}
        assert not live & given
        assert [int(x) for x in table[1][sorted(live)]] == [pages[i] for i in sorted(live)]
        assert len({pages[i] for i in live}) == len(live), "a page twice"
        length += m
        assert c.length(s) == length and len(pages) - len(c._gone[s]) + c.free_pages == 40
        assert len(pages) - len(c._gone[s]) <= (window + sinks + 17) // 16 + 4
    assert len(c._pages[s]) > 150
    c.free(s)
    assert c.free_pages == 40
