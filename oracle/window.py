"""Windowed attention over a paged cache and multi-axis rotary positions, in float64 NumPy.

The masking, tables and contexts are those of the reference's attention
(src/paged_kv_serving/engine/attention.py:42-121), with the window and the sinks added.
"""

from __future__ import annotations

import numpy as np

__all__ = ["axis_of_frequency", "visible_keys", "window_attention"]


def visible_keys(position: int, context: int, window: int, sinks: int) -> np.ndarray:
    """The key positions a row sees."""
    keys = np.arange(max(0, min(context, position + 1)))
    return keys[(keys > position - window) | (keys < sinks)]


def window_attention(
    queries, positions, seqs, key_cache, value_cache, tables, contexts, scale, window: int, sinks: int
) -> tuple[np.ndarray, np.ndarray]:
    """Output ``[T, heads, dim]`` and, for error bounds, the largest ``scale * sum |q k|`` of each
    (row, head). Padding rows (a sequence outside the tables) are NaN; blocks outside the pool are
    skipped."""
    queries = np.asarray(queries, np.float64)
    total, heads, dim = queries.shape
    blocks, block, kv_heads, _ = key_cache.shape
    out = np.full(queries.shape, np.nan)
    size = np.zeros((total, heads))
    for t in range(total):
        if not 0 <= seqs[t] < len(contexts):
            continue
        keys = visible_keys(int(positions[t]), int(contexts[seqs[t]]), window, sinks)
        ids = np.asarray(tables[seqs[t]])[keys // block]
        inside = (ids >= 0) & (ids < blocks)
        ids, keys = ids[inside], keys[inside]
        k = np.asarray(key_cache[ids, keys % block], np.float64)
        v = np.asarray(value_cache[ids, keys % block], np.float64)
        for h in range(heads):
            g = h // (heads // kv_heads)
            if keys.size == 0:
                out[t, h] = 0.0
                continue
            score = scale * (k[:, g] @ queries[t, h])
            size[t, h] = abs(scale) * (np.abs(k[:, g]) @ np.abs(queries[t, h])).max()
            p = np.exp(score - score.max())
            out[t, h] = (p @ v[:, g]) / p.sum()
    return out, size


def axis_of_frequency(sections, interleaved: bool) -> list[int]:
    """The position axis that turns each frequency."""
    if not interleaved:
        return [axis for axis, count in enumerate(sections) for _ in range(count)]
    axes = len(sections)
    return [i % axes if i < axes * sections[i % axes] else 0 for i in range(sum(sections))]
