"""The windowed attention oracle against closed forms and the causal oracle, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.window import axis_of_frequency, visible_keys, window_attention


def test_visible_keys_by_their_definition() -> None:
    assert visible_keys(9, 10, 4, 0).tolist() == [6, 7, 8, 9]
    assert visible_keys(9, 10, 4, 2).tolist() == [0, 1, 6, 7, 8, 9]
    assert visible_keys(9, 10, 4, 7).tolist() == list(range(10))  # the sinks meet the window
    assert visible_keys(9, 10, 100, 0).tolist() == list(range(10))
    assert visible_keys(9, 5, 4, 1).tolist() == [0]  # past the context: only the sink is left
    assert visible_keys(9, 0, 4, 1).tolist() == visible_keys(-1, 10, 4, 1).tolist() == []


def make(rows, context, heads, kv_heads, dim, block, seed):
    rng = np.random.default_rng(seed)
    blocks = -(-context // block)
    table = rng.permutation(blocks + 2)[:blocks][None]
    pools = [rng.standard_normal((blocks + 2, block, kv_heads, dim)) for _ in range(2)]
    return rng.standard_normal((rows, heads, dim)), np.arange(context - rows, context), pools, table


@pytest.mark.parametrize("context,block", [(1, 1), (7, 3), (40, 16)])
def test_a_wide_window_is_causal_attention(context, block) -> None:
    q, positions, (keys, values), table = make(min(5, context), context, 2, 2, 4, block, context)
    got, _ = window_attention(q, positions, np.zeros(len(q), int), keys, values, table, [context], 0.5, context, 0)
    flat = [pool[table[0]].reshape(-1, 2, 4)[:context] for pool in (keys, values)]
    for t, p in enumerate(positions):
        scores = 0.5 * np.einsum("hd,khd->hk", q[t], flat[0][: p + 1])
        weights = np.exp(scores - scores.max(1, keepdims=True))
        want = np.einsum("hk,khd->hd", weights / weights.sum(1, keepdims=True), flat[1][: p + 1])
        assert np.allclose(got[t], want, rtol=1e-12, atol=1e-12)


def test_a_window_of_one_returns_the_own_value_and_heads_share_keys() -> None:
    q, positions, (keys, values), table = make(6, 20, 6, 2, 4, 8, 3)
    got, _ = window_attention(q, positions, np.zeros(6, int), keys, values, table, [20], 0.5, 1, 0)
    flat = values[table[0]].reshape(-1, 2, 4)
    for t, p in enumerate(positions):
        for h in range(6):
            assert np.allclose(got[t, h], flat[p, h // 3])


def test_padding_empty_rows_and_blocks_outside_the_pool() -> None:
    q, positions, (keys, values), table = make(3, 12, 2, 1, 4, 4, 5)
    positions = np.asarray([-1, 11, 11])
    got, size = window_attention(q, positions, [0, 7, 0], keys, values, table, [12], 0.5, 5, 1)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and (size >= 0).all()
    holes = table.copy()
    holes[0, 0] = -3  # the sink's block: only the window is left
    some, _ = window_attention(q, positions, [0, 7, 0], keys, values, holes, [12], 0.5, 5, 1)
    want, _ = window_attention(q, positions, [0, 7, 0], keys, values, table, [12], 0.5, 5, 0)
    assert np.array_equal(some[2], want[2])


def test_a_planted_mistake_is_seen() -> None:
    q, positions, (keys, values), table = make(3, 12, 2, 1, 4, 4, 6)
    args = (q, positions, np.zeros(3, int), keys, values, table, [12], 0.5)
    right, _ = window_attention(*args, 5, 1)
    for window, sinks in ((4, 1), (6, 1), (5, 0), (5, 2)):
        assert np.abs(window_attention(*args, window, sinks)[0] - right).max() > 1e-3


def test_axes_of_frequencies() -> None:
    assert axis_of_frequency((2, 1, 3), False) == [0, 0, 1, 2, 2, 2]
    assert axis_of_frequency((2, 2, 2), True) == [0, 1, 2, 0, 1, 2]
    assert axis_of_frequency((4, 1, 1), True) == [0, 1, 2, 0, 0, 0]
    assert axis_of_frequency((5,), True) == [0] * 5
