"""Sampling by its definition, in float64 NumPy: temperature, top-k, min-p and top-p as cuts of one
order (falling logit, equal ones by id), and a draw with a given uniform number.

Extends the reference's sampling (src/paged_kv_serving/engine/sampling.py:28-74).
"""

from __future__ import annotations

import numpy as np

__all__ = ["sample_row"]


def sample_row(
    logits: np.ndarray, uniform: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0
) -> int:
    """The token of one row; the settings are float32 values."""
    logits = np.asarray(logits, dtype=np.float64)
    if np.isnan(logits).any():
        return int(np.flatnonzero(np.isnan(logits))[0])
    top = logits.max()
    if not temperature > 0 or top == -np.inf:
        return int(logits.argmax())
    order = np.lexsort((np.arange(logits.size), -logits))
    x = logits[order]
    with np.errstate(invalid="ignore"):
        weights = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / np.float64(np.float32(temperature)))))
    if top == np.inf:
        weights = (x == top).astype(np.float64)
    kept = int(np.count_nonzero((weights >= np.float64(np.float32(min_p))) & (weights > 0)))
    kept = max(1, kept if top_k <= 0 else min(kept, top_k))
    mass = np.cumsum(weights[:kept])
    last = kept - 1
    if top_p < 1:
        last = min(last, int(np.searchsorted(mass, np.float64(np.float32(top_p)) * mass[-1], side="left")))
    drawn = int(np.searchsorted(mass, np.float64(np.float32(uniform)) * mass[last], side="right"))
    return int(order[min(drawn, last)])
