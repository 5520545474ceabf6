"""A serving step's metadata from its requests' lengths, request by request in plain Python.

Slots and positions are those of the reference's batches (src/paged_kv_serving/engine/runner.py:149-159, 184-212).
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np

__all__ = ["step_metadata"]


def step_metadata(query_lens, context_lens, tables, free, next_free: int, block_size: int, num_rows: int) -> SimpleNamespace:
    """The result, with ``tables`` a changed copy; ``served`` says which requests were."""
    tables = np.array(tables, np.int64)
    query_seq, positions, slots = [-1] * num_rows, [0] * num_rows, [-1] * num_rows
    next_free = min(max(next_free, 0), len(free))
    starts, contexts, served = [0], [], []
    row = asked = taken = 0
    for i, (q, c) in enumerate(zip(query_lens, context_lens)):
        q, c = max(int(q), 0), int(c)
        first, row = row, row + q
        starts.append(min(row, num_rows))
        sound = c >= q and c <= tables.shape[1] * block_size and row <= num_rows
        held, used = (-(-(c - q) // block_size), -(-c // block_size)) if sound else (0, 0)
        asked += used - held
        if not sound or (used > held and asked > len(free) - next_free):
            contexts.append(max(c - q, 0))
            served.append(False)
            continue
        for k in range(held, used):
            tables[i, k] = free[next_free + taken]
            taken += 1
        contexts.append(c)
        served.append(True)
        for k in range(q):
            position = c - q + k
            block = tables[i, position // block_size]
            query_seq[first + k], positions[first + k] = i, position
            if block >= 0:
                slots[first + k] = block * block_size + position % block_size
    return SimpleNamespace(query_seq=query_seq, query_positions=positions, positions=positions, slot_mapping=slots, query_starts=starts,
                           context_lens=contexts, next_free=[next_free + taken], tables=tables, served=served)  # fmt: skip
