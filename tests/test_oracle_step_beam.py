"""The oracles of step metadata and beam search against closed forms, invariants and brute force, on the CPU."""

from __future__ import annotations

import itertools
import math

import numpy as np
import pytest

from oracle.beam import reorder_group, select_group
from oracle.step import step_metadata


def test_a_step_by_hand() -> None:
    """Two requests: one with a full block and one more token, a new one of five; blocks of four."""
    tables = [[7, 0, 0], [0, 0, 0]]
    s = step_metadata([1, 5], [5, 5], tables, [3, 9, 4, 1], 1, 4, 8)
    assert s.query_seq == [0, 1, 1, 1, 1, 1, -1, -1]
    assert s.positions == [4, 0, 1, 2, 3, 4, 0, 0]
    assert s.slot_mapping == [36, 16, 17, 18, 19, 4, -1, -1]
    assert s.query_starts == [0, 1, 6] and s.context_lens == [5, 5] and s.next_free == [4]
    assert s.tables.tolist() == [[7, 9, 0], [4, 1, 0]]


@pytest.mark.parametrize("change,served", [
    ({}, [True, True, True]), ({"free": [5, 6]}, [True, True, False]), ({"free": [5]}, [True, False, False]), ({"free": []}, [False, False, False]),
    ({"num_rows": 9}, [True, True, False]), ({"context_lens": [4, 30, 6]}, [True, False, True]), ({"context_lens": [4, 1, 6]}, [True, False, True]),
    ({"query_lens": [0, 2, 6]}, [True, True, True]), ({"query_lens": [0, 2, 6], "free": []}, [True, False, False]),
], ids=str)  # fmt: skip
def test_requests_that_cannot_be_served(change, served) -> None:
    """Blocks of four: the requests need 1, 1 and 2 of the free ones."""
    args = dict(query_lens=[3, 2, 6], context_lens=[4, 5, 6], tables=np.zeros((3, 4)), free=[5, 6, 7, 8], next_free=0, block_size=4, num_rows=11)
    if change.get("query_lens"):
        change = {**change, "context_lens": [4, 5, 6]}
    args |= change
    if "query_lens" not in change:
        args["context_lens"] = [3, *args["context_lens"][1:]]
    s = step_metadata(**args)
    assert s.served == served
    for i, (ok, q, c) in enumerate(zip(served, args["query_lens"], args["context_lens"])):
        assert s.query_seq.count(i) == (q if ok else 0)
        assert s.context_lens[i] == (c if ok else max(c - q, 0))
        assert ok or not s.tables[i].any()


def test_a_decode_loop_fills_its_blocks_in_order() -> None:
    tables, next_free = np.zeros((2, 5), np.int64), 0
    for step in range(1, 18):
        s = step_metadata([1, 1], [step, step], tables, list(range(20, 40)), next_free, 4, 2)
        tables, next_free = s.tables, s.next_free[0]
    assert tables.tolist() == [[20, 22, 24, 26, 28], [21, 23, 25, 27, 29]] and next_free == 10


def brute(logits, scores, count):
    """Every continuation's score by its definition."""
    every = []
    for b, row in enumerate(logits):
        total = sum(math.exp(x) for x in row)
        every += [(scores[b] + math.log(math.exp(x) / total), b, v) for v, x in enumerate(row)]
    return sorted(every, key=lambda e: -e[0])[:count]


@pytest.mark.parametrize("beams,vocab,count", [(1, 5, 3), (3, 7, 4), (4, 3, 12)])
def test_selection_against_brute_force(beams, vocab, count) -> None:
    rng = np.random.default_rng(beams)
    logits, scores = rng.standard_normal((beams, vocab)), -rng.random(beams)
    for (score, beam, token), (want, b, v) in zip(select_group(logits, scores, count), brute(logits, scores, count)):
        assert (beam, token) == (b, v) and abs(score - want) < 1e-12


def test_ties_ended_and_dead_beams() -> None:
    flat = np.zeros((2, 4))
    assert [e[1:] for e in select_group(flat, [0.0, 0.0], 8)] == [(b, t) for b in (0, 1) for t in range(4)]
    assert [e[1:] for e in select_group(flat, [-1.0, 0.0], 5)] == [(1, 0), (1, 1), (1, 2), (1, 3), (0, 0)]
    # Ended beams go on with the end token at their score, whatever their rows hold.
    got = select_group(np.full((2, 4), np.nan), [-3.0, -2.0], 3, [True, True], 9)
    assert got == [(-2.0, 1, 9), (-3.0, 0, 9), (-math.inf, 0, 9)]
    for bad in (np.nan, np.inf):
        rows = np.zeros((2, 4))
        rows[0, 2] = bad
        assert [e[1:] for e in select_group(rows, [0.0, -5.0], 5, end_token=1)] == [(1, 0), (1, 1), (1, 2), (1, 3), (0, 1)]
    only = np.full((1, 4), -np.inf)
    assert select_group(only, [0.0], 2) == [(-math.inf, 0, 0)] * 2
    only[0, 3] = -2.0
    assert select_group(only, [-1.0], 2, end_token=3) == [(-1.0, 0, 3), (-math.inf, 0, 3)]
    assert select_group(flat, [-math.inf, math.nan], 1) == [(-math.inf, 0, 0)]


@pytest.mark.parametrize("beams", [1, 2, 3, 4])
def test_every_reordering_keeps_every_childs_contents(beams) -> None:
    """For all parents: after the copies, at once or in any order, a child's table reads what its parent's read."""
    block = 4
    tables = np.concatenate([np.full((beams, 1), 90), np.arange(beams * 3).reshape(beams, 3)], axis=1)  # one shared block
    for parents in itertools.product(range(beams), repeat=beams):
        for context in (5, 7, 8, 12, 13, 16):
            new, copies = reorder_group(tables, parents, context, block)
            contents = {b: b for b in [90, *range(beams * 3)]}
            sources, targets = [c[0] for c in copies], [c[1] for c in copies]
            assert len(set(targets)) == len(targets) and not set(sources) & set(targets)
            contents |= {t: s for s, t in copies}
            used = -(-context // block)
            for child, parent in enumerate(parents):
                assert [contents[b] for b in new[child, :used]] == tables[parent, :used].tolist()
                assert new[child, used:].tolist() == tables[child, used:].tolist()
            if context % block:  # last blocks stay the rows' own, and only the group's are used
                assert sorted(new[:, used - 1]) == sorted(tables[:, used - 1])
                assert len(copies) == beams - len(set(parents))
            else:
                assert not copies


def test_parents_outside_the_group_and_contexts_outside_the_table() -> None:
    tables = np.arange(6).reshape(2, 3)
    assert reorder_group(tables, [-1, 2], 5, 4)[0].tolist() == tables.tolist()
    assert reorder_group(tables, [1, 1], 100, 4) == (pytest.approx(np.asarray([[3, 4, 5], [3, 4, 5]])), [])
    assert reorder_group(tables, [1, 1], -3, 4)[0].tolist() == tables.tolist()
