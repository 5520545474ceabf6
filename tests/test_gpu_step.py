"""step_metadata against the plain definition: requests of any lengths, few free blocks, padding, captured growth."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.step import step_metadata

pytestmark = pytest.mark.gpu


def requests(seqs, most_query, most_context, block, width, seed, extra=20):
    """Requests with blocks for what they have cached, and a list of free ones."""
    rng = np.random.default_rng(seed)
    query = rng.integers(0, most_query + 1, seqs)
    before = rng.integers(0, most_context, seqs)
    before[rng.random(seqs) < 0.3] = 0
    held = -(-before // block)
    need = int((-(-(before + query) // block) - held).sum())
    ids = rng.permutation(int(held.sum()) + need + extra)
    tables = rng.integers(0, 100, (seqs, width))  # past what a request has: anything
    at = 0
    for i, n in enumerate(held):
        tables[i, :n] = ids[at : at + n][:width]
        at += n
    return {"query_lens": query, "context_lens": before + query, "tables": tables, "free": ids[at:], "next_free": 0, "block_size": block,
            "num_rows": int(query.sum())}  # fmt: skip


def put(x, device):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device)


def call(device, d, **more):
    from paged_kv_serving_amd import ops

    tables = put(d["tables"], device)
    step = ops.step_metadata(put(d["query_lens"], device), put(d["context_lens"], device), tables, put(d["free"], device), put([d["next_free"]], device),
                             block_size=d["block_size"], num_rows=d["num_rows"], **more)  # fmt: skip
    return step, tables


def check(device, d, **more):
    step, tables = call(device, d, **more)
    want = step_metadata(**d)
    for name in step._fields:
        got = getattr(step, name)
        assert got.dtype.is_signed and got.is_contiguous()
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(getattr(want, name)).reshape(got.shape), err_msg=name)
    np.testing.assert_array_equal(tables.cpu().numpy(), want.tables)
    return want


@pytest.mark.parametrize("block", [1, 3, 16, 64])
@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 511, 512, 513, 1300])
def test_requests_of_many_lengths(device, seqs, block):
    for most_query, most_context in ((1, 200), (3, 50), (200, 500) if seqs < 200 else (9, 500)):
        d = requests(seqs, most_query, most_context, block, -(-(most_query + most_context) // block), seqs + block)
        assert all(check(device, d).served)
        check(device, {**d, "num_rows": d["num_rows"] + 37})


@pytest.mark.parametrize("seqs", [5, 700])
def test_requests_that_cannot_be_served(device, seqs):
    d = requests(seqs, 40, 300, 16, 22, seqs, extra=0)
    free = len(d["free"])
    for few in (0, 1, free // 3, free - 1, free):
        want = check(device, {**d, "free": d["free"][:few]})
        assert all(want.served) == (few == free)
    for rows in (0, 1, d["num_rows"] // 2, d["num_rows"] - 1):
        assert not all(check(device, {**d, "num_rows": rows}).served)
    rng = np.random.default_rng(1)
    bad = {name: d[name].copy() for name in ("query_lens", "context_lens")}
    bad["context_lens"][rng.random(seqs) < 0.3] = 16 * 22 + 1  # too wide
    bad["context_lens"][rng.random(seqs) < 0.1] = -5
    bad["query_lens"][rng.random(seqs) < 0.1] = -(2**31)
    bad["context_lens"][-1], bad["query_lens"][-1] = 2**31 - 1, 2**31 - 1
    assert not all(check(device, {**d, **bad}).served)


def test_where_the_free_list_stands(device):
    d = requests(30, 5, 60, 8, 9, 3, extra=50)
    for next_free in (0, 1, 17, len(d["free"]) - 1, len(d["free"]), len(d["free"]) + 5, -3):
        check(device, {**d, "next_free": next_free})
    empty = {**d, "free": np.zeros(0, np.int64)}
    check(device, empty)


def test_negative_table_entries_have_no_slot(device):
    d = requests(20, 6, 60, 8, 9, 4)
    d["tables"][::2, 0] = -1
    check(device, d)


def test_nothing_to_do_and_an_earlier_result(device):
    from paged_kv_serving_amd import ops

    d = requests(0, 1, 1, 16, 4, 0)
    check(device, {**d, "num_rows": 0})
    check(device, {**d, "num_rows": 5})
    d = requests(40, 20, 90, 16, 8, 1)
    first, _ = call(device, requests(40, 20, 90, 16, 8, 1))
    for seed in (2, 3):
        e = {**requests(40, 20, 90, 16, 8, seed), "num_rows": d["num_rows"]}
        check(device, e, out=first)
    check(device, {**requests(7, 1, 9, 16, 8, 1), "tables": np.zeros((7, 0)), "num_rows": 4})  # tables without a column
    assert ops.MAX_STEP_ROWS == 1 << 21


def test_a_captured_step_whose_requests_grow(device):
    """One graph replayed: contexts, tables and the free list move on the device alone."""
    import torch

    from paged_kv_serving_amd import ops

    seqs, block, width = 6, 4, 16
    rng = np.random.default_rng(0)
    contexts = rng.integers(1, 20, seqs)
    held = -(-contexts // block)
    ids = rng.permutation(200)
    tables = np.zeros((seqs, width), np.int64)
    for i, n in enumerate(held):
        tables[i, :n] = ids[int(held[:i].sum()) :][:n]
    free = ids[int(held.sum()) :]
    q, c, t, f, at = (put(x, device) for x in (np.ones(seqs), contexts, tables, free, [0]))
    out = ops.step_metadata(q, c, t, f, at, block_size=block, num_rows=seqs + 2)
    t.copy_(put(tables, device))

    def run():
        c.add_(1)
        ops.step_metadata(q, c, t, f, at, block_size=block, num_rows=seqs + 2, out=out)
        at.copy_(out.next_free)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    next_free = 0
    for step in range(12):
        if step == 5:  # the host changes what a replay sees: a request that waits
            q[2:3].zero_()
        graph.replay()
        torch.cuda.synchronize()
        contexts = contexts + 1
        query = np.ones(seqs) if step < 5 else np.asarray([1, 1, 0, 1, 1, 1])
        want = step_metadata(query, contexts, tables, free, next_free, block, seqs + 2)
        tables, next_free = want.tables, want.next_free[0]
        for name in out._fields:
            np.testing.assert_array_equal(getattr(out, name).cpu().numpy().ravel(), np.asarray(getattr(want, name)).ravel(), err_msg=name)
        np.testing.assert_array_equal(t.cpu().numpy(), tables)


def test_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
    good = dict(query_lens=i32(3), context_lens=i32(3), block_tables=i32(3, 4), free_blocks=i32(5), next_free=i32(1), block_size=16, num_rows=6)
    out = ops.step_metadata(**good)
    assert ops.step_metadata(**{**good, "next_free": None}).next_free.item() == 0
    bad = [
        {"query_lens": i32(3).long()}, {"query_lens": i32(3, 1)}, {"context_lens": i32(2)}, {"context_lens": i32(3).float()}, {"block_tables": i32(2, 4)},
        {"block_tables": i32(3, 4).long()}, {"block_tables": i32(4, 3).t()}, {"free_blocks": i32(5).long()}, {"free_blocks": i32(10)[::2]}, {"next_free": i32(2)},
        {"next_free": i32(1).long()}, {"block_size": 0}, {"block_size": 1 << 30}, {"num_rows": -1}, {"num_rows": (1 << 21) + 1}, {"query_lens": i32(3).cpu()},
        {"out": out._replace(positions=out.query_positions)}, {"out": out._replace(query_starts=i32(3))}, {"out": out._replace(slot_mapping=out.slot_mapping.cpu())},
    ]  # fmt: skip
    for change in bad:
        with pytest.raises(ValueError):
            ops.step_metadata(**{**good, **change})
    with pytest.raises(ValueError, match="own"):
        ops.step_metadata(**{**good, "out": out, "next_free": out.next_free})
    with pytest.raises(ValueError, match="own"):
        ops.step_metadata(**{**good, "out": out, "context_lens": out.context_lens})


def test_outputs_in_the_memory_of_an_input_are_refused(device):
    """Parts of one buffer: each output over each input and, where the inputs lie apart, the same result as from buffers of their own."""
    import torch

    from paged_kv_serving_amd import ops

    room = torch.zeros(400, dtype=torch.int32, device=device)
    room[:8] = torch.tensor([1, 2, 0, 3, 5, 17, 30, 3], dtype=torch.int32)
    query, context, free, next_free = room[:4], room[4:8], room[8:20], room[20:21]
    free.copy_(torch.arange(12, dtype=torch.int32))
    tables = torch.arange(100, 112, dtype=torch.int32, device=device).view(4, 3)
    want_tables = tables.clone()
    want = ops.step_metadata(query.clone(), context.clone(), want_tables, free.clone(), next_free.clone(), block_size=16, num_rows=8)
    wide = room[24:88].view(torch.int64)
    out = ops.StepMetadata(room[100:108], room[108:116], wide[:8], wide[8:16], room[116:121], room[121:125], room[125:126])
    got = ops.step_metadata(query, context, tables, free, next_free, block_size=16, num_rows=8, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(tables, want_tables)
    for name, size in (("query_seq", 8), ("query_positions", 8), ("query_starts", 5), ("context_lens", 4), ("next_free", 1)):
        for first in (0, 3, 7, 19, 20):  # over the lengths, the list of free blocks, its place
            with pytest.raises(ValueError, match="own inputs"):
                ops.step_metadata(query, context, tables, free, next_free, block_size=16, num_rows=8, out=out._replace(**{name: room[first : first + size]}))
    with pytest.raises(ValueError, match="own inputs"):
        ops.step_metadata(query, context, room[10:22].view(4, 3), free, next_free, block_size=16, num_rows=8)
    same = context.clone()  # one tensor as two inputs: prompts without a cached token
    both = ops.step_metadata(same, same, tables.clone(), free, block_size=16, num_rows=60)
    apart = ops.step_metadata(same, same.clone(), tables.clone(), free, block_size=16, num_rows=60)
    assert all(torch.equal(a, b) for a, b in zip(both, apart))
