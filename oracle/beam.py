"""Beam search by its definition, in float64 NumPy: the best continuations of a group, and what becomes of its rows' blocks.

The reference samples one sequence (src/paged_kv_serving/engine/sampling.py:28-74) and copies blocks on the host
(src/paged_kv_serving/engine/runner.py:128-133).
"""

from __future__ import annotations

import math

import numpy as np

__all__ = ["reorder_group", "select_group"]


def select_group(logits, scores, count: int, finished=None, end_token: int = 0) -> list[tuple[float, int, int]]:
    """``count`` (score, beam, token) of one group of beams, best first."""
    found = []
    for beam, (row, score) in enumerate(zip(np.asarray(logits, np.float64), np.asarray(scores, np.float64))):
        if not math.isfinite(score):
            continue
        if finished is not None and finished[beam]:
            found.append((-score, beam, 0.0, end_token))
            continue
        most = row.max()
        if not math.isfinite(most):  # a NaN, +inf, or nothing above -inf
            continue
        norm = math.log(math.fsum(np.exp(row - most)))
        # No token outside a row's best `count`, ties by number, can be among the group's.
        order = np.lexsort((np.arange(row.size), -row))[:count]
        found += [(-(score + ((row[token] - most) - norm)), beam, -row[token], int(token)) for token in order if row[token] > -math.inf]
    best = [(-negative, beam, token) for negative, beam, _, token in sorted(found)[:count]]
    return best + [(-math.inf, 0, end_token)] * (count - len(best))


def reorder_group(tables, parents, context: int, block_size: int) -> tuple[np.ndarray, list[tuple[int, int]]]:
    """One group's new tables ``[beams, blocks]`` and its block copies (source, target)."""
    tables = np.asarray(tables)
    beams, width = tables.shape
    parents = [p if 0 <= p < beams else child for child, p in enumerate(parents)]
    full, part = divmod(min(max(context, 0), width * block_size), block_size)
    idle = [row for row in range(beams) if row not in parents]
    new, copies, named = tables.copy(), [], set()
    for child, parent in enumerate(parents):
        new[child, :full] = tables[parent, :full]
        if part:
            keeper = idle.pop(0) if parent in named else parent
            new[child, full] = tables[keeper, full]
            if keeper != parent:
                copies.append((int(tables[parent, full]), int(tables[keeper, full])))
        named.add(parent)
    return new, copies
