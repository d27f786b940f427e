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
