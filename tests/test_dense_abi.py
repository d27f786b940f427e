"""Host-side checks of the dense attention, paged cache and axes entry points: every call
here fails validation or is an empty no-op, so nothing is launched and no pointer is
dereferenced (sections, which is host memory, is real)."""

import ctypes
import os

import pytest
import torch

import ssa_amd
from ssa_amd import _lib

FAKE = ctypes.c_void_p(1 << 20)
MISALIGNED = ctypes.c_void_p((1 << 20) + 8)
OK, INVALID, UNSUPPORTED, WORKSPACE = (_lib.SSA_OK, _lib.SSA_ERR_INVALID_ARGUMENT, _lib.SSA_ERR_UNSUPPORTED,
                                       _lib.SSA_ERR_WORKSPACE)


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libssa_hip.so not built (run __graft_entry__.build())")
    return _lib.load()


def _call(L, name, defaults, kw):
    a = {**defaults, **kw}
    assert set(a) == set(defaults)
    st = getattr(L, name)(*a.values())
    return st, (L.ssa_last_error() or b"").decode()


SPANS = dict(starts=FAKE, docs=3, prefix=FAKE, batch=2, n=100, n_q=100, q_pos0=0, causal=1, spans=FAKE, stream=None)
HEADS = dict(dtype=_lib.DTYPE_BF16, batch=1, n=1000, n_q=1000, q_pos0=0, h_q=8, h_kv=2, d=64)
ROWS = {f"{x}_{s}": v for x in "qkv" for s, v in (("sb", 64000 * 8), ("sn", 512), ("sh", 64))}
FORWARD = dict(q=FAKE, k=FAKE, v=FAKE, **HEADS, **ROWS, spans=None, scale=8.0, cap=0.0, slopes=None, out=FAKE, o_sb=0,
               o_sn=512, o_sh=64, out_low=None, lse=None, ws=FAKE, ws_bytes=1 << 30, stream=None)
BACKWARD = dict(q=FAKE, k=FAKE, v=FAKE, **HEADS, **ROWS, spans=None, scale=8.0, cap=0.0, slopes=None, out=FAKE,
                out_low=None, o_sb=0, o_sn=512, o_sh=64, dout=FAKE, do_sb=0, do_sn=512, do_sh=64, lse=FAKE, dq=FAKE, dk=FAKE, dv=FAKE,
                ws=FAKE, ws_bytes=1 << 30, stream=None)
PAGED = dict(q=FAKE, k=FAKE, v=FAKE, dtype=_lib.DTYPE_BF16, tokens=10, batch=3, h_q=8, h_kv=2, d=64, q_st=512, q_sh=64,
             k_st=128, k_sh=64, v_st=128, v_sh=64, k_pages=FAKE, v_pages=FAKE, num_pages=100, page_size=16, kp_sp=2048,
             kp_st=128, kp_sh=64, vp_sp=2048, vp_st=128, vp_sh=64, table=FAKE, table_stride=64, max_pages=64, starts=FAKE,
             cached=FAKE, max_new=8, max_len=1000, scale=8.0, cap=0.0, slopes=None, out=FAKE, o_st=512, o_sh=64, flag=None,
             ws=FAKE, ws_bytes=1 << 30, stream=None)
SECTIONS = (ctypes.c_int32 * 4)(8, 12, 12, 0)
NEGATIVE = (ctypes.c_int32 * 4)(33, -1, 0, 0)
AXES = dict(q=FAKE, k=FAKE, dtype=_lib.DTYPE_BF16, batch=1, n=100, h_q=8, h_k=2, d=64, q_sb=0, q_sn=512, q_sh=64, k_sb=0,
            k_sn=128, k_sh=64, pos=FAKE, pos_dtype=_lib.INDEX_I64, p_sa=100, p_sb=100, axes=3, sections=SECTIONS, freqs=FAKE,
            rot=64, inverse=0, q_out=FAKE, qo_sb=0, qo_sn=512, qo_sh=64, k_out=FAKE, ko_sb=0, ko_sn=128, ko_sh=64,
            stream=None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(n=-1), INVALID, "shape"), (dict(docs=0), INVALID, "docs"), (dict(starts=None), INVALID, "one document"),
    (dict(spans=None), INVALID, "null"), (dict(n=1 << 31), INVALID, "shape"), (dict(batch=0, spans=None), OK, ""),
])
def test_mask_spans(L, kw, status, text):
    st, msg = _call(L, "ssa_mask_spans", SPANS, kw)
    assert st == status and (st == OK or text in msg), msg


DENSE = [
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(h_q=9), INVALID, "divisible"), (dict(h_q=34), UNSUPPORTED, "group"),
    (dict(d=60), UNSUPPORTED, "head_dim"), (dict(d=136), UNSUPPORTED, "head_dim"), (dict(d=0), INVALID, "shape"),
    (dict(n=-1), INVALID, "shape"), (dict(q_pos0=-1), INVALID, "shape"), (dict(n=1 << 31), UNSUPPORTED, "2^31"),
    (dict(n_q=1 << 29), UNSUPPORTED, "2^31"), (dict(scale=0.0), INVALID, "scale"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(cap=-1.0), INVALID, "softcap"),
    (dict(cap=float("nan")), INVALID, "softcap"), (dict(q=None), INVALID, "null"), (dict(v=None), INVALID, "null"),
    (dict(out=None), INVALID, "null"), (dict(q_sn=1 << 23 | 8), UNSUPPORTED, "strides"), (dict(q_sh=-64), UNSUPPORTED, "strides"),
    (dict(q=MISALIGNED), UNSUPPORTED, "q must"), (dict(k_sn=516), UNSUPPORTED, "k must"),
    (dict(v_sh=4), UNSUPPORTED, "v must"), (dict(o_sn=4), UNSUPPORTED, "out must"),
    (dict(batch=0, q=None), OK, ""),
]


@pytest.mark.parametrize("kw,status,text", DENSE + [
    (dict(n_q=4, ws=None), WORKSPACE, "workspace"), (dict(n_q=4, ws_bytes=100), WORKSPACE, "workspace"),
    (dict(n_q=4, ws=MISALIGNED), INVALID, "workspace"), (dict(n_q=0, q=None), OK, ""),
])
def test_masked_attention(L, kw, status, text):
    if "ws" in kw or "ws_bytes" in kw:
        assert L.ssa_masked_attention_workspace_bytes(_lib.DTYPE_BF16, 1, 4000, 4, 8, 2, 64) > 100
        kw = {**kw, "n": 4000}
    st, msg = _call(L, "ssa_masked_attention", FORWARD, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("kw,status,text", DENSE + [
    (dict(ws=None), WORKSPACE, "workspace"), (dict(ws_bytes=100), WORKSPACE, "workspace"),
    (dict(ws=MISALIGNED), INVALID, "workspace"), (dict(lse=None), INVALID, "null"), (dict(dk=None), INVALID, "null"),
    (dict(do_sn=4), UNSUPPORTED, "dout must"), (dict(dv=MISALIGNED), UNSUPPORTED, "dv must"),
    (dict(n_q=0), INVALID, "no gradient"),
])
def test_masked_attention_backward(L, kw, status, text):
    st, msg = _call(L, "ssa_masked_attention_backward", BACKWARD, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("kw,status,text", [x for x in DENSE if not {"n", "n_q", "q_pos0", "q_sn", "k_sn", "o_sn", "batch"} & set(x[0])] + [
    (dict(tokens=-1), INVALID, "shape"), (dict(page_size=24), UNSUPPORTED, "page_size"),
    (dict(page_size=4), UNSUPPORTED, "page_size"), (dict(page_size=8192), UNSUPPORTED, "page_size"),
    (dict(tokens=1 << 30), UNSUPPORTED, "2^31"), (dict(max_pages=1 << 28), UNSUPPORTED, "2^31"),
    (dict(max_new=0), INVALID, "max_new"), (dict(num_pages=0), INVALID, "num_pages"), (dict(k=None), INVALID, "null"),
    (dict(table=None), INVALID, "null"), (dict(kp_st=4), UNSUPPORTED, "k_pages"), (dict(vp_sp=4), UNSUPPORTED, "v_pages"),
    (dict(k_st=4), UNSUPPORTED, "k must"), (dict(ws=None), WORKSPACE, "workspace"),
    (dict(ws=MISALIGNED), INVALID, "workspace"), (dict(tokens=0, q=None), OK, ""), (dict(batch=0, q=None), OK, ""),
])
def test_paged_step(L, kw, status, text):
    st, msg = _call(L, "ssa_paged_step", PAGED, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(pos_dtype=5), INVALID, "positions"), (dict(h_q=0), INVALID, "shape"),
    (dict(rot=63), INVALID, "rot"), (dict(rot=66), INVALID, "rot"), (dict(h_k=5000), UNSUPPORTED, "4096"), (dict(axes=0), UNSUPPORTED, "axes"),
    (dict(axes=5), UNSUPPORTED, "axes"), (dict(sections=None), INVALID, "null"), (dict(axes=2), INVALID, "sections"),
    (dict(sections=NEGATIVE), INVALID, "negative"), (dict(rot=32), INVALID, "sections"), (dict(freqs=None), INVALID, "null"),
    (dict(k=None), INVALID, "null"), (dict(q_out=None), INVALID, "null"), (dict(n=0, q=None), OK, ""),
])
def test_rope_axes(L, kw, status, text):
    st, msg = _call(L, "ssa_rope_axes", AXES, kw)
    assert st == status and (st == OK or text in msg), msg


@pytest.mark.parametrize("max_new,max_len,max_pages", [(8, 1000, 64), (8, 1025, 64), (1 << 62, 1025, 64), (10, 70000, 64),
                                                       (1, 1 << 30, 8), (300, 1024, 1)])
@pytest.mark.parametrize("tokens,batch", [(10, 3), (300, 1), (700, 16)])
def test_paged_workspace_of_any_bounds(L, max_new, max_len, max_pages, tokens, batch):
    """Bounds past the tokens and the table are allowed; the call needs what the sizes say."""
    need = L.ssa_paged_step_workspace_bytes(_lib.DTYPE_BF16, tokens, batch, 8, 2, 64, max_new, max_len)
    kw = dict(tokens=tokens, batch=batch, max_new=max_new, max_len=max_len, max_pages=max_pages)
    if need == 0:
        return
    for ws, have in ((FAKE, need - 1), (None, need)):
        st, msg = _call(L, "ssa_paged_step", PAGED, dict(kw, ws=ws, ws_bytes=have))
        assert st == WORKSPACE and f"workspace of {need} bytes" in msg, msg


def test_cache_refuses_pages_that_no_step_takes():
    for page in (0, 4, 24, 8192):
        with pytest.raises(ValueError, match="page_size"):
            ssa_amd.PagedKVCache(4, page, 2, 64, device="cpu")
    for d in (0, 12, 136):
        with pytest.raises(ValueError, match="head_dim"):
            ssa_amd.PagedKVCache(4, 16, 2, d, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        ssa_amd.PagedKVCache(4, 16, 2, 64, dtype=torch.float16, device="cpu")


def test_python_refuses_gradients_it_does_not_have():
    q = torch.zeros(1, 4, 2, 8, requires_grad=True)
    with pytest.raises(NotImplementedError, match="slopes"):
        ssa_amd.masked_attention(q, q, q, slopes=torch.ones(2, requires_grad=True))
    with pytest.raises(NotImplementedError, match="freqs"):
        ssa_amd.rope_axes(q, q, torch.zeros(1, 1, 4, dtype=torch.int32), ssa_amd.axis_rope_freqs(8).requires_grad_(True), (4,))


def test_python_refuses_host_tensors():
    q = torch.zeros(1, 4, 2, 8)
    ints = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.masked_attention(q, q, q)
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.mask_spans(4, 1, device="cpu")
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.mask_spans(4, 1, doc_starts=ints)
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.paged_step(q[0], q[0], q[0], q, q, ints, ints[0], ints[0])
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.rope_axes(q, q, ints[None], ssa_amd.axis_rope_freqs(8), (4,))
    with pytest.raises(ValueError, match="prefix_lens"):
        ssa_amd.mask_spans(4, 1, causal=False, prefix_lens=ints)


def test_heads_far_apart(L):
    """Head strides are 64-bit: what refuses these calls is the missing workspace.  The backward
    wants a group's heads within 2 GiB."""
    far = {f"{x}_sh": 1 << 33 for x in "qkv"}
    st, msg = _call(L, "ssa_masked_attention", FORWARD, dict(far, n=4000, n_q=4, o_sh=1 << 33, ws=None))
    assert st == WORKSPACE, msg
    st, msg = _call(L, "ssa_paged_step", PAGED, dict({f"{x}_sh": 1 << 33 for x in ("q", "k", "v", "kp", "vp", "o")}, ws=None))
    assert st == WORKSPACE, msg
    room = (0x7FFFFFF0 // 2 - 64 - 32 * 512) // 3  # g = 4: 32 tokens and 3 heads from the tile's first row
    for x in ("q", "do"):
        st, msg = _call(L, "ssa_masked_attention_backward", BACKWARD, {f"{x}_sh": room // 8 * 8, "ws": None})
        assert st == WORKSPACE, msg
        st, msg = _call(L, "ssa_masked_attention_backward", BACKWARD, {f"{x}_sh": room // 8 * 8 + 8, "ws": None})
        assert st == UNSUPPORTED and "2 GiB" in msg, msg
    st, msg = _call(L, "ssa_masked_attention_backward", BACKWARD, dict(h_q=2, q_sh=1 << 40, do_sh=1 << 40, ws=None))
    assert st == WORKSPACE, msg


def test_paged_step_zeroed(L):
    for kw, status, text in ((dict(batch=0), INVALID, "sequence"), (dict(tokens=0, batch=0, q=None), OK, ""),
                             (dict(out=None), INVALID, "null"), (dict(ws=None), WORKSPACE, "ssa_paged_step_zeroed: workspace")):
        st, msg = _call(L, "ssa_paged_step_zeroed", PAGED, kw)
        assert st == status and (st == OK or text in msg), msg


def test_python_refuses_tangents_that_it_would_drop():
    """Forward-mode differentiation, with and without gradients enabled."""
    import torch.autograd.forward_ad as fwd
    from ssa_amd.ssa_layer import rope_rows

    x = torch.zeros(1, 4, 2, 8)
    ints = torch.zeros(1, 4, dtype=torch.int32)
    freqs = ssa_amd.axis_rope_freqs(8)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        slopes = fwd.make_dual(torch.ones(2), torch.ones(2))
        calls = [lambda: ssa_amd.masked_attention(dual, x, x), lambda: ssa_amd.masked_attention(x, x, dual),
                 lambda: ssa_amd.masked_attention(x, x, x, slopes=slopes),
                 lambda: ssa_amd.rope_axes(dual, None, ints[None], freqs, (4,)), lambda: ssa_amd.rope_axes(x, dual, ints[None], freqs, (4,)),
                 lambda: ssa_amd.rope_axes(x, x, ints[None], fwd.make_dual(freqs, freqs), (4,)),
                 lambda: ssa_amd.paged_step(x[0], dual[0], x[0], x, x, ints, ints[0], ints[0]),
                 lambda: ssa_amd.paged_step(x[0], None, None, x, dual, ints, ints[0], ints[0]),
                 lambda: rope_rows(dual, x[0, 0], x[0, 0], 8, True)]
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled):
                for call in calls:
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call()
        with pytest.raises(RuntimeError, match="HIP"):  # (no tangent: the device is what is wrong)
            ssa_amd.masked_attention(x, x, x)


def test_python_refuses_half_precision_beside_other_types():
    x = torch.zeros(1, 4, 2, 8, dtype=torch.float16)
    for other in (x.float(), x.bfloat16()):
        for args in ((x, other, other), (x, x, other), (x, other, x)):
            with pytest.raises(TypeError, match="share a dtype"):
                ssa_amd.masked_attention(*args)


def test_paged_step_refuses_gradients_it_does_not_have():
    """With gradients enabled only: under no_grad it goes on to the next check, the device."""
    x = torch.zeros(4, 2, 8)
    ints = torch.zeros(1, 4, dtype=torch.int32)
    args = dict(q=x, k=x, v=x, k_pages=x[None], v_pages=x[None], table=ints, starts=ints[0], cached=ints[0], slopes=torch.ones(2))
    for name in ("q", "k", "v", "k_pages", "v_pages", "slopes"):
        leaf = {**args, name: args[name].clone().requires_grad_(True)}
        with pytest.raises(NotImplementedError, match="no gradient"):
            ssa_amd.paged_step(**leaf)
        with torch.no_grad(), pytest.raises(RuntimeError, match="HIP"):
            ssa_amd.paged_step(**leaf)
    with pytest.raises(RuntimeError, match="HIP"):
        ssa_amd.paged_step(**args)
    cache = ssa_amd.PagedKVCache(8, 8, 2, 8, dtype=torch.float32, device="cpu")
    seq = cache.add()
    with pytest.raises(NotImplementedError, match="no gradient"):
        cache.step(x.clone().requires_grad_(True), x, x, [seq], [4])
    assert cache.free_pages == 8 and cache.length(seq) == 0


@pytest.mark.parametrize("name,args", [("ssa_masked_attention", FORWARD), ("ssa_masked_attention_backward", BACKWARD),
                                       ("ssa_paged_step", PAGED)])
def test_scales_and_caps_that_fp32_does_not_hold(L, name, args):
    """1 / (scale cap) and a score times it have to be fp32 numbers of full precision."""
    for kw in (dict(cap=3e38), dict(cap=1e-40), dict(scale=1e-31), dict(scale=1e31), dict(scale=1e20, cap=1e11), dict(scale=1e-20, cap=1e-11)):
        st, msg = _call(L, name, args, kw)
        assert st == INVALID and "range" in msg, msg
    tight = {} if name != "ssa_masked_attention" else dict(n=4000, n_q=4)
    for kw in (dict(cap=1e29), dict(cap=2e-30), dict(scale=2e-30), dict(scale=9e29), dict(scale=1e20, cap=1e-30)):
        st, msg = _call(L, name, args, {**tight, **kw, "ws": None})
        assert st == WORKSPACE, msg


def test_workspaces_of_sizes_that_no_call_takes(L):
    """Products of the sizes overflow; a batch of 2^62 on 4 heads would divide by 0, and as many
    tokens in groups of 4 would count as none."""
    huge = 1 << 62
    st, msg = _call(L, "ssa_paged_step", PAGED, dict(tokens=huge))
    assert st == UNSUPPORTED and "2^31" in msg, msg
    for a in ((10, huge, 8, 4, 64, 8, 1000), (huge, 3, 8, 4, 64, 8, 1000), (10, 3, 8, 4, 64, 8, (1 << 63) - 1)):
        assert L.ssa_paged_step_workspace_bytes(_lib.DTYPE_BF16, *a) == 0
    for name in ("ssa_masked_attention_workspace_bytes", "ssa_masked_attention_backward_workspace_bytes"):
        for B, n, n_q in ((huge, 100, 100), (1, huge, 4), (1, 100, huge)):
            assert getattr(L, name)(_lib.DTYPE_BF16, B, n, n_q, 8, 4, 64) == 0
