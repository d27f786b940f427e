"""rope_axes against its formula in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _turned(x, pos, freqs, sections, sign=1.0):
    """x [B, n, h, d] turned in 64 bits, pair by pair."""
    x = x.double()
    y = x.clone()
    half = freqs.shape[0]
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    for m in range(half):
        ang = sign * (pos[axis[m]].double() * float(freqs[m]))[..., None]
        y[..., m] = x[..., m] * ang.cos() - x[..., half + m] * ang.sin()
        y[..., half + m] = x[..., half + m] * ang.cos() + x[..., m] * ang.sin()
    return y


def _check(got, x, want, half, what):
    """The cosine and sine are within 2^-23 (their argument's and polynomial's roundings, each
    2^-25 and less, and the last one's), the two products and the sum round to fp32, the result
    once more to its type."""
    r = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24
    x = x.double().abs()
    mag = x.clone()
    mag[..., :half] += x[..., half:2 * half]
    mag[..., half:2 * half] += x[..., :half]
    bound = r * want.abs() + 2.0 ** -21.5 * mag
    got = got.detach().cpu().double()
    assert ((got - want).abs() <= bound).all(), (what, float(((got - want).abs() / bound.clamp(min=1e-30)).max()))


CASES = [
    # dtype, B, n, h_q, h_k, d, sections, position dtype
    (BF16, 1, 1, 4, 2, 64, (8, 12, 12), torch.int64),
    (F32, 2, 7, 3, 1, 64, (8, 8), torch.int32),
    (BF16, 2, 33, 8, 2, 128, (16, 24, 24), torch.int64),
    (F32, 1, 100, 5, 5, 80, (10, 15, 15), torch.int32),
    (BF16, 1, 65, 4, 1, 96, (20,), torch.int64),
    (BF16, 1, 50, 2, 2, 20, (1, 0, 2, 4), torch.int32),
    (F32, 1, 41, 2, 1, 10, (5, 0), torch.int64),
    (BF16, 3, 700, 28, 4, 128, (16, 24, 24), torch.int64),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("far", [0, 10 ** 6, 2 ** 31 - 2000])
def test_values_and_gradients(dev, case, far):
    from ssa_amd import axis_rope_freqs, rope_axes

    dtype, B, n, h_q, h_k, d, sections, pdt = case
    g = torch.Generator().manual_seed(50)
    q, k, dq, dk = (torch.randn(B, n, h, d, generator=g).to(dtype) for h in (h_q, h_k, h_q, h_k))
    pos = (torch.randint(-900, 900, (len(sections), B, n), generator=g) + far).to(pdt)
    half = sum(sections)
    freqs = axis_rope_freqs(2 * half, 1e4)
    print(f"axes {case} {far}", flush=True)
    leaves = [q.to(dev).requires_grad_(True), k.to(dev).requires_grad_(True)]
    out = rope_axes(*leaves, pos.to(dev), freqs.to(dev), sections)
    grads = torch.autograd.grad(out, leaves, (dq.to(dev), dk.to(dev)))
    for name, got, x, sign in (("q", out[0], q, 1.0), ("k", out[1], k, 1.0), ("dq", grads[0], dq, -1.0), ("dk", grads[1], dk, -1.0)):
        assert got.dtype == dtype
        _check(got, x, _turned(x, pos, freqs, sections, sign), half, name)
    only = rope_axes(leaves[0], None, pos.to(dev), freqs.to(dev), sections)
    assert torch.equal(only, out[0])
    assert torch.equal(torch.autograd.grad(only, leaves[0], dq.to(dev))[0], grads[0])


def test_gradient_against_differences(dev):
    from ssa_amd import axis_rope_freqs, rope_axes

    g = torch.Generator().manual_seed(51)
    q, way, dq = (torch.randn(1, 9, 2, 16, generator=g).to(dev) for _ in range(3))
    pos = torch.randint(0, 500, (2, 1, 9), generator=g).to(dev)
    freqs = axis_rope_freqs(16, 1e4, dev)
    leaf = q.clone().requires_grad_(True)
    grad = torch.autograd.grad(rope_axes(leaf, None, pos, freqs, (3, 5)), leaf, dq)[0]
    ends = [(rope_axes(q + s * way, None, pos, freqs, (3, 5)).double() * dq).sum() for s in (1, -1)]
    # the rotation is linear: the difference is exact up to fp32 roundings of 288 products
    mag = float((way.abs() * dq.abs()).sum())
    assert abs(float((ends[0] - ends[1]) / 2 - (grad.double() * way).sum())) < 2.0 ** -19 * (mag + float((q.abs() * dq.abs()).sum())) * 2


def test_second_order(dev):
    """The backward is a rotation itself: its gradient is the rotation."""
    from ssa_amd import axis_rope_freqs, rope_axes

    g = torch.Generator().manual_seed(53)
    q, k, a, b = (torch.randn(1, 6, 2, 16, generator=g).to(dev).requires_grad_(True) for _ in range(4))
    pos = torch.randint(0, 500, (2, 1, 6), generator=g).to(dev)
    freqs = axis_rope_freqs(16, 1e4, dev)
    x, y = rope_axes(q, k, pos, freqs, (3, 5))
    dq, dk = torch.autograd.grad((x, y), (q, k), (a, b), create_graph=True)
    u, w = torch.randn_like(q), torch.randn_like(k)
    da, db = torch.autograd.grad((dq, dk), (a, b), (u, w))
    ru, rw = rope_axes(u, w, pos, freqs, (3, 5))
    assert torch.equal(da, ru) and torch.equal(db, rw)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(x, q, a)
    z = rope_axes(q, None, pos, freqs, (3, 5))
    dq = torch.autograd.grad(z, q, a, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad(dq, a, u)[0], rope_axes(u, None, pos, freqs, (3, 5)))


def test_layouts_streams_graph(dev):
    from ssa_amd import axis_rope_freqs, rope_axes

    g = torch.Generator().manual_seed(52)
    q, k = (torch.randn(2, 45, h, 64, generator=g).to(BF16).to(dev) for h in (4, 2))
    pos = torch.randint(0, 300, (3, 45), generator=g).to(dev)
    freqs, sections = axis_rope_freqs(48, 1e6, dev), (8, 8, 8)
    want = rope_axes(q, k, pos, freqs, sections)
    full = pos[:, None].expand(3, 2, 45)
    for a, b in ((q.transpose(1, 2).contiguous().transpose(1, 2), k), (q, torch.nn.functional.pad(k, (3, 2))[..., 3:67]),
                 (torch.cat((q, q), -1)[..., :64], k.transpose(2, 3).contiguous().transpose(2, 3))):
        for p in (full, full.contiguous(), pos.t().contiguous().t()):
            got = rope_axes(a, b, p, freqs, sections)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = rope_axes(q[1], k[1], pos, freqs, sections)
    assert torch.equal(one[0], want[0][1]) and torch.equal(one[1], want[1][1])
    half = rope_axes(q.half(), None, pos, freqs, sections)
    assert half.dtype == torch.float16
    assert torch.equal(half, rope_axes(q.float(), None, pos, freqs, sections).half())
    # several axes at one position are one axis: ssa_rope with tables of the same angles
    from ssa_amd import kernels

    same = torch.arange(45, device=dev).expand(3, 2, 45)
    ang = torch.arange(45, device=dev, dtype=torch.float64)[:, None] * freqs
    ang = torch.cat((ang, ang), -1)
    ref = kernels.rope(q.float(), ang.cos().float(), ang.sin().float(), 48, by_head=False)
    got = rope_axes(q.float(), None, same, freqs, sections)
    assert (got - ref).abs().max() < 2.0 ** -20 * q.abs().max()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope_axes(q, k, pos, freqs, sections)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        cap = rope_axes(q, k, pos, freqs, sections)
    for _ in range(3):
        pos.add_(11)
        graph.replay()
        torch.cuda.synchronize()
        eager = rope_axes(q, k, pos, freqs, sections)
        assert torch.equal(cap[0], eager[0]) and torch.equal(cap[1], eager[1])


def test_empty_and_rejects(dev):
    from ssa_amd import axis_rope_freqs, rope_axes

    q, pos, freqs = torch.zeros(1, 5, 2, 16, device=dev), torch.zeros(2, 1, 5, device=dev, dtype=torch.int64), axis_rope_freqs(16, device=dev)
    assert rope_axes(q[:, :0], None, pos[..., :0], freqs, (4, 4)).shape == (1, 0, 2, 16)
    for change, err, text in (((q, None, pos, freqs, (4, 5)), RuntimeError, "sections"), ((q, None, pos, freqs, (9, -1)), RuntimeError, "section"),
                              ((q, None, pos, freqs.float(), (4, 4)), TypeError, "float64"),
                              ((q, None, pos.float(), freqs, (4, 4)), TypeError, "indices|positions"),
                              ((q, None, pos[:1], freqs, (4, 4)), ValueError, "positions"),
                              ((q, q[:, :4], pos, freqs, (4, 4)), ValueError, "go with"),
                              ((q[..., :8], None, pos, freqs, (4, 4)), RuntimeError, "rot"),
                              ((q.cpu(), None, pos, freqs, (4, 4)), RuntimeError, "HIP"),
                              ((q, None, torch.zeros(5, 1, 5, device=dev, dtype=torch.int64), freqs, (2, 2, 2, 1, 1)), NotImplementedError, "axes")):
        with pytest.raises(err, match=text):
            rope_axes(*change)
