"""Score caps of any size, against the 64-bit oracle: c tanh(s / c) keeps s as c grows."""

import pytest
import torch

from tests.dense_oracle import attend, check, spans_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# Up to a cap of 1024 the bf16 kernels may be off by cap 2^-22 (the oracle's own bound is twice
# that), beyond it by 2^-20 of the score; the fp32 kernels' tanh by a few 2^-24 of it.
CAPS = [(1024.0, None), (1030.0, 2.0 ** -20), (1e5, 2.0 ** -20), (1e6, 2.0 ** -20), (1e12, 2.0 ** -20),
        (5e28, 2.0 ** -20), (1e-30, None)]


def _inputs(seed, dtype, n_q, n, h_q, h_kv, d):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(1, m, h, d, generator=g).to(dtype) for m, h in ((n_q, h_q), (n, h_kv), (n, h_kv), (n_q, h_q))]


@pytest.mark.parametrize("dtype,n_q,n,d", [(F32, 37, 37, 64), (BF16, 37, 37, 64), (BF16, 37, 37, 128), (BF16, 3, 900, 64)], ids=str)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap,rel", CAPS)
def test_masked(dev, dtype, n_q, n, d, bias, cap, rel):
    from ssa_amd import masked_attention

    q, k, v, dout = _inputs(61, dtype, n_q, n, 4, 2, d)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0]) if bias else None
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = masked_attention(*leaves, softcap=cap, slopes=None if slopes is None else slopes.to(dev))
    res = (out, *torch.autograd.grad(out, leaves, dout.to(dev)))
    want = attend(q[0], k[0], v[0], spans_of(n, n_q, n - n_q), cap, slopes, n - n_q, dout[0], cap_rel=rel)
    for got, name in zip(res, ("out", "dq", "dk", "dv")):
        check(got[0], *want[name], f"{name}, cap {cap}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("m", [1, 70])
@pytest.mark.parametrize("cap,rel", CAPS)
def test_paged(dev, dtype, m, cap, rel):
    from ssa_amd import paged_step

    n, h_q, h_kv, d, page = 130, 4, 2, 64, 16
    q, k, v, _ = _inputs(62, dtype, m, n, h_q, h_kv, d)
    pages = -(-n // page)
    pools = []
    for t in (k, v):
        pool = torch.zeros(pages * page, h_kv, d, dtype=dtype)
        pool[:n] = t[0]
        pools.append(pool.view(pages, page, h_kv, d).to(dev))
    ints = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([list(range(pages))], [0, m], [n - m])]
    out = paged_step(q[0].to(dev), None, None, *pools, *ints, softcap=cap, check=True)
    check(out, *attend(q[0], k[0], v[0], spans_of(n, m, n - m), cap, None, n - m, cap_rel=rel)["out"], f"cap {cap}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_a_cap_that_no_score_reaches_changes_nothing_but_roundings(dev, dtype):
    """Two keys, whose weights show the scores: c tanh(s / c) is s to 2^-36 for c = 1e6 (and
    |s| below 10), and the oracle's (d + 20) 2^-24 of a score holds the cap's 2^-20 as well."""
    from ssa_amd import masked_attention

    q, k, v, _ = _inputs(63, dtype, 2, 2, 1, 1, 64)
    for slopes in (None, torch.zeros(1, device=dev)):
        out = masked_attention(q.to(dev), k.to(dev), v.to(dev), softcap=1e6, slopes=slopes)
        check(out[0], *attend(q[0], k[0], v[0], spans_of(2, 2, 0), 0.0, None, 0)["out"], "against no cap")
