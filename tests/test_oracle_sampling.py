"""The sampling oracle against hand-made rows and its frequencies, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.sampling import sample_row

#: Weights 1, 1/2, 1/4, 1/4 at ids 2, 0, 3, 1: together 2, in units of an eighth 4, 2, 1, 1.
ROW = np.log(np.asarray([0.5, 0.25, 1.0, 0.25]))


@pytest.mark.parametrize("uniform,token", [(0.0, 2), (0.49, 2), (0.51, 0), (0.74, 0), (0.76, 1), (0.86, 1), (0.88, 3), (0.999, 3)])
def test_tokens_by_cumulative_mass(uniform, token) -> None:
    assert sample_row(ROW, uniform) == token


def test_the_cuts() -> None:
    assert [sample_row(ROW, u, top_k=2) for u in (0.0, 0.6, 0.7, 0.999)] == [2, 2, 0, 0]
    assert [sample_row(ROW, u, min_p=0.4) for u in (0.0, 0.6, 0.7, 0.999)] == [2, 2, 0, 0]
    assert [sample_row(ROW, u, top_p=0.45) for u in (0.0, 0.999)] == [2, 2]
    assert [sample_row(ROW, u, top_p=0.7) for u in (0.0, 0.6, 0.7, 0.999)] == [2, 2, 0, 0]
    # top-p counts the mass that top-k leaves: 2 / 3 of it is the first token's.
    assert [sample_row(ROW, u, top_k=2, top_p=0.6) for u in (0.0, 0.999)] == [2, 2]
    assert sample_row(ROW, 0.999, top_k=3) == 1  # of equal logits the lower id stays
    assert sample_row(ROW, 0.999, min_p=1.0) == 2


def test_temperature() -> None:
    assert sample_row(ROW, 0.999, temperature=0.0) == 2
    # At half the temperature the weights are squared: 16, 4, 1, 1 of 22.
    assert [sample_row(ROW, u, temperature=0.5) for u in (0.72, 0.74, 0.90, 0.92, 0.99)] == [2, 0, 0, 1, 3]


def test_special_rows() -> None:
    inf, nan = np.inf, np.nan
    assert sample_row([0.0, nan, 5.0, nan], 0.9) == 1
    assert sample_row([-inf, -inf], 0.9) == 0
    assert [sample_row([-inf, 1.0, -inf], u) for u in (0.0, 0.999)] == [1, 1]
    assert [sample_row([3.0, inf, 0.0, inf], u) for u in (0.0, 0.49, 0.51, 0.999)] == [1, 1, 3, 3]
    assert sample_row([7.0], 0.5) == 0


def test_frequencies_are_the_probabilities() -> None:
    rng = np.random.default_rng(1)
    logits = rng.standard_normal(12)
    tokens = [sample_row(logits, (i + 0.5) / 4000) for i in range(4000)]  # every quantile once
    p = np.exp(logits) / np.exp(logits).sum()
    assert np.abs(np.bincount(tokens, minlength=12) / 4000 - p).max() <= 1 / 4000


def test_a_planted_mistake_is_seen() -> None:
    rng = np.random.default_rng(2)
    logits = rng.standard_normal(50)
    right = [sample_row(logits, i / 64, top_k=20, top_p=0.9) for i in range(64)]
    for wrong in ({"top_k": 20}, {"top_p": 0.9, "top_k": 3}, {"top_k": 20, "top_p": 0.9, "temperature": 1.2}):
        assert [sample_row(logits, i / 64, **wrong) for i in range(64)] != right
