"""The 8-bit cache's oracle against torch's own conversion, closed forms and invariants, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import e4m3

ALL = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
FINITE = np.unique(ALL[np.isfinite(ALL)])


def test_every_code_is_its_own_nearest_and_ties_go_to_even() -> None:
    assert FINITE.size == 253 and FINITE.max() == e4m3.LARGEST and FINITE[FINITE > 0].min() == 2.0**-9
    assert np.array_equal(e4m3.nearest(FINITE), FINITE)
    middle = (FINITE[1:] + FINITE[:-1]) / 2
    down, up = e4m3.nearest(np.nextafter(middle, -np.inf)), e4m3.nearest(np.nextafter(middle, np.inf))
    assert np.array_equal(down, FINITE[:-1]) and np.array_equal(up, FINITE[1:])
    tied = e4m3.nearest(middle)
    codes = torch.from_numpy(tied).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (codes % 2 == 0).all()


def test_nearest_is_the_conversion_of_torch() -> None:
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(200_000) * np.exp2(rng.integers(-14, 8, 200_000))).astype(np.float32)
    x = x[np.abs(x) <= e4m3.LARGEST]
    assert np.array_equal(e4m3.nearest(x), torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy().astype(np.float64))
    assert np.isnan(e4m3.nearest([np.inf, -np.inf, np.nan])).all()


@pytest.mark.parametrize("most,scale", [(448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (3.5, 2.0**-7), (3.50001, 2.0**-6), (0.0, 2.0**-100),
                                        (1e-30, 2.0**-100), (2.0**120, 2.0**112)])  # fmt: skip
def test_block_scale(most, scale) -> None:
    assert e4m3.block_scale(most) == scale


def pools(blocks=4, block=4, heads=2, dim=8):
    return np.zeros((blocks, block, heads, dim)), np.zeros((blocks, heads))


def test_tokens_one_by_one_and_together() -> None:
    """Where values do not fall below 2^-6 of the format, a block filled token by token is the block filled at once."""
    rng = np.random.default_rng(1)
    new = rng.uniform(0.5, 8.0, (16, 2, 8)) * rng.choice([-1, 1], (16, 2, 8))
    together, apart = pools(), pools()
    e4m3.append(*together, new, np.arange(16))
    for t in range(16):
        e4m3.append(*apart, new[t : t + 1], [t])
    assert np.array_equal(together[1], apart[1])
    assert np.array_equal(together[0], apart[0])
    off = np.abs(e4m3.values(*together).reshape(16, 2, 8) - new)
    assert (off <= 2.0**-4 * np.abs(new)).all()


def test_a_scale_grows_with_its_block_and_starts_anew() -> None:
    codes, scales = pools()
    small, large = np.full((1, 2, 8), 0.01), np.full((1, 2, 8), 100.0)
    e4m3.append(codes, scales, small, [4])
    first = scales[1].copy()
    e4m3.append(codes, scales, large, [5])
    assert (scales[1] > first).all() and (scales[1] == e4m3.block_scale(100.0)).all()
    assert np.abs(e4m3.values(codes, scales)[1, 0] - 0.01).max() <= 2.0**-10 * scales[1, 0]  # half of the smallest step
    e4m3.append(codes, scales, small, [6])
    assert (scales[1] == e4m3.block_scale(100.0)).all()  # it does not shrink
    e4m3.append(codes, scales, small, [4])
    assert np.array_equal(scales[1], first)  # written from its first place: anew
    assert (scales[[0, 2, 3]] == 0).all()


def test_padding_bad_values_and_an_empty_call() -> None:
    codes, scales = pools()
    e4m3.append(codes, scales, np.ones((3, 2, 8)), [-1, 16, 1 << 40])
    assert not codes.any() and not scales.any()
    e4m3.append(codes, scales, np.ones((0, 2, 8)), [])
    new = np.ones((2, 2, 8))
    new[0, 0, 3], new[1, 1, 0] = np.inf, np.nan
    e4m3.append(codes, scales, new, [0, 1])
    assert np.isnan(codes[0, 0, 0, 3]) and np.isnan(codes[0, 1, 1, 0]) and np.isnan(codes).sum() == 2
    assert (scales[0] == e4m3.block_scale(1.0)).all()


def test_a_planted_mistake_is_seen() -> None:
    """A scale of one power of two less overflows, one of two more loses a bit of small values."""
    x = np.asarray([448.0 * 0.9, 1.3 * 2.0**-7])
    right = e4m3.block_scale(np.abs(x).max())
    assert np.isfinite(e4m3.nearest(x / right)).all() and not np.isfinite(e4m3.nearest(x / (right / 2))).all()
    assert e4m3.nearest(x[1] / (4 * right)) * 4 * right != e4m3.nearest(x[1] / right) * right
