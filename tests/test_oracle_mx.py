"""The microscaled oracle (oracle/mx.py) pinned against library casts, brute force and written-out grids."""
import numpy as np
import pytest
import torch

from oracle import mx


def test_grids():
    assert mx.code_values("e2m1")[:8].tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    got = mx.code_values("e4m3")
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)]) and np.isnan(got[[127, 255]]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_scale_is_the_smallest_that_fits(fmt):
    bits = torch.arange(0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)   # every finite magnitude
    x = torch.zeros(len(bits), 32, dtype=torch.bfloat16)
    x[:, 7] = -bits
    b = mx.scale_bytes(x.double().numpy(), fmt)[:, 0].astype(np.int64)
    a, m = bits.double().numpy(), mx.LARGEST[fmt]
    assert (a <= m * np.exp2(b - 127.0)).all()
    assert ((a > m * np.exp2(b - 128.0)) | (b == 0)).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_codes_are_nearest_with_ties_to_even(fmt):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 64, generator=g) * torch.exp2(torch.randint(-6, 7, (64, 64), generator=g).float())).to(torch.bfloat16)
    codes, b = mx.quantise(x, fmt)
    s = np.exp2(b.numpy().astype(float) - 127).repeat(32, -1)
    y = x.double().numpy() / s
    grid = mx.code_values(fmt)
    half = len(grid) // 2
    ok = np.flatnonzero(np.isfinite(grid[:half]))
    dist = np.abs(np.abs(y)[..., None] - grid[:half][ok])
    best = dist.min(-1)
    c = codes.numpy().astype(np.int64) & (half - 1)
    assert np.array_equal(np.take_along_axis(dist, c[..., None], -1)[..., 0], best)
    ties = (dist == best[..., None]).sum(-1) == 2
    assert (c[ties] % 2 == 0).all()
    assert np.array_equal((codes.numpy() & half) != 0, np.signbit(y))
    if fmt == "e4m3":
        assert np.array_equal(codes.numpy(), torch.from_numpy(y).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_values_round_trip_and_are_bf16(fmt):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(33, 128, generator=g).to(torch.bfloat16)
    codes, b = mx.quantise(x, fmt)
    v = mx.values(mx.pack(codes, fmt), b, fmt)
    assert torch.equal(v.to(torch.bfloat16).double(), v)
    # half a step of the code's grid: 2^-4 of the value, or half the smallest step (E2M1: 2^-2, at most 1/4 of the scale), and no
    # value is clipped
    s = torch.exp2(b.double() - 127).repeat_interleave(32, -1)
    bound = torch.maximum(v.abs() * (2.0 ** -4 if fmt == "e4m3" else 0.25), s * (2.0 ** -10 if fmt == "e4m3" else 0.25))
    assert ((v - x.double()).abs() <= bound).all()
    again, b2 = mx.quantise(v.to(torch.bfloat16), fmt)
    assert torch.equal(mx.values(mx.pack(again, fmt), b2, fmt), v)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_non_finite_blocks_are_nan(fmt):
    x = torch.ones(3, 96, dtype=torch.bfloat16)
    x[0, 5], x[1, 40], x[2, 95] = float("inf"), float("nan"), float("-inf")
    codes, b = mx.quantise(x, fmt)
    assert (b == 255).tolist() == [[True, False, False], [False, True, False], [False, False, True]]
    v = mx.values(mx.pack(codes, fmt), b, fmt)
    assert torch.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all() and torch.isnan(v[1, 32:64]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_finite_rows_have_finite_bf16_values(fmt):
    """Every finite bf16 as the largest of its block: the value is a finite bf16, and no code that stands for one is nearer."""
    bits = torch.arange(0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(len(bits), 32, dtype=torch.bfloat16)
    x[:, 7] = -bits
    codes, b = mx.quantise(x, fmt)
    v = mx.values(mx.pack(codes, fmt), b, fmt)
    assert torch.isfinite(v).all() and torch.equal(v.to(torch.bfloat16).double(), v)
    grid = mx.code_values(fmt)[:len(mx.code_values(fmt)) // 2]
    stands_for = torch.from_numpy(grid[np.isfinite(grid)])[None] * torch.exp2(b.double() - 127)      # [rows, codes]
    stands_for[~torch.isfinite(stands_for.to(torch.bfloat16))] = float("inf")
    best = (stands_for - bits.double()[:, None]).abs().min(-1).values
    assert torch.equal((v[:, 7] + bits.double()).abs(), best)
