"""paged_read's rounding and what rows without a key hold, bit by bit."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4M3 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def nearest_bf16(x):
    """float64 to bfloat16 in one rounding, ties to even (torch goes by way of float32): for a value between
    2^e and 2^(e + 1) a multiple of 2^(e - 7), of 2^-133 below the smallest normal one."""
    e = torch.frexp(x)[1].double().clamp(min=-125) - 1  # (frexp: a value in [0.5, 1) times 2^e)
    step = torch.exp2(e - 7)
    y = (x / step).round() * step
    return torch.where(torch.isfinite(x), y, x).float().to(BF16)


def test_nearest_bf16():
    """The reference itself, on the host's grid of values: what a bfloat16 holds stays, ties go to even."""
    grid = torch.arange(0, 0x7F80, dtype=torch.int16).view(BF16).double()
    assert torch.equal(nearest_bf16(grid).double(), grid)
    mid = (grid[1:] + grid[:-1]) / 2
    even = torch.where(torch.arange(len(mid)) % 2 == 0, grid[:-1], grid[1:])
    assert torch.equal(nearest_bf16(mid).double(), even)
    for way in (grid[1:], grid[:-1]):
        assert torch.equal(nearest_bf16(torch.nextafter(mid, way)).double(), way)


@pytest.mark.parametrize("hold", [I8, E4M3])
def test_codes_are_read_in_one_rounding(dev, hold):
    from ssa_amd import paged_read

    g = torch.Generator().manual_seed(81)
    T, h, d, page = 4096, 2, 128, 16
    codes = torch.randint(-128, 128, (2, T, h, d), generator=g).to(I8)
    if hold == E4M3:
        codes = torch.where(codes.view(E4M3).float().isnan(), 3, codes)
    scales = torch.exp2(torch.rand(2, T, h, generator=g) * 12 - 9)
    scales[:, 0] = 0.022805606946349144
    codes[:, 0, :, 0] = 17
    scales[:, 1], scales[:, 2], scales[:, 3], scales[:, 4], scales[:, 5] = 2.0 ** -126, 1.3e-42, 3.1e36, math.nan, 0.0
    pools = [x.view(hold).view(-1, page, h, d).to(dev) for x in codes]
    both = [x.view(-1, page, h).to(dev) for x in scales]
    at = dict(table=torch.arange(T // page, device=dev, dtype=torch.int32)[None],
              starts=torch.tensor([0, T], device=dev, dtype=torch.int32), first=torch.zeros(1, device=dev, dtype=torch.int32))
    exact = codes.view(hold).float().double() * scales.double()[..., None]
    for dtype, want in ((BF16, nearest_bf16(exact)), (F32, exact.float())):
        got = paged_read(*pools, tokens=T, dtype=dtype, k_scales=both[0], v_scales=both[1], check=True, **at)
        for x, y in zip(got, want):
            x = x.cpu()
            assert torch.equal(x.isnan(), y.isnan()) and torch.equal(torch.nan_to_num(x, nan=0.0), torch.nan_to_num(y, nan=0.0))
    if hold == I8:
        assert float(exact[0, 0, 0, 0]) == 17 * float(torch.tensor(0.022805606946349144))
        assert float(nearest_bf16(exact)[0, 0, 0, 0]) == 0.388671875
    assert not torch.equal(torch.nan_to_num(nearest_bf16(exact)), torch.nan_to_num(exact.float().to(BF16))), "no product tells them apart"
