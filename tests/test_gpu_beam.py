"""beam_select and beam_reorder against the float64 definitions: vocabularies of any length, ties, ended and dead beams,
masked rows, every kind of parents and states."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle.beam import reorder_group, select_group

pytestmark = pytest.mark.gpu


def select(device, logits, scores, beams, count, finished=None, end_token=0, **more):
    import torch

    from paged_kv_serving_amd import ops

    more = {"finished": None if finished is None else torch.as_tensor(np.asarray(finished, bool)).to(device), "end_token": end_token, **more}
    return ops.beam_select(logits.to(device), torch.as_tensor(np.asarray(scores, np.float32)).to(device), num_beams=beams, count=count, **more)


def check(device, logits, scores, beams, count, finished=None, end_token=0, near=False, **more):
    """Beams and tokens are the definition's. A score is a number within 2^-36 (1 + |logits|) of the definition's (sums and
    exponentials to 2^-40, a logarithm, two additions of double numbers), rounded once to float32. ``near``: two scores that the
    definition has within twice 2^-36 (1 + |score|) of each other may come in either order, since each is within that of the exact
    one (the largest logit is taken from the logit first, which rounds that difference alone): rows with the same sum of
    exponentials in another order have sums that differ in their last bits."""
    best = select(device, logits, scores, beams, count, finished, end_token, **more)
    got = [x.cpu().numpy() for x in best]
    rows = logits.float().numpy().astype(np.float64)
    scores = np.asarray(scores, np.float32).astype(np.float64).ravel()
    for g in range(len(rows) // beams):
        at = slice(g * beams, (g + 1) * beams)
        want = select_group(rows[at], scores[at], count, None if finished is None else np.asarray(finished).ravel()[at], end_token)
        chosen = [(int(b), int(t)) for b, t in zip(got[1][g], got[2][g])]
        if near:
            score_of = {(b, t): s for s, b, t in select_group(rows[at], scores[at], 4 * count, None, end_token)}
            assert len(set(chosen)) == count, f"group {g}"
            for pair, (score, _, _) in zip(chosen, want):
                assert abs(score_of[pair] - score) <= 2 * 2.0**-36 * (1 + abs(score)), f"group {g}"
        else:
            assert chosen == [(b, t) for _, b, t in want], f"group {g}"
        largest = np.abs(rows[at][np.isfinite(rows[at])]).max(initial=0.0)
        for x, (score, _, _) in zip(got[0][g].astype(np.float64), want):
            assert x == score or abs(x - score) <= 2.0**-24 * abs(score) + 2.0**-36 * (1 + largest), (g, x, score)
    return best


def rows_of(groups, beams, vocab, io, seed, sharp=2.0):
    import torch

    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn((groups * beams, vocab), generator=gen) * sharp).to(getattr(torch, io))
    return logits, -10 * torch.rand(groups * beams, generator=gen).numpy()


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 500, 2048, 2049, 8191, 8193, 50257])
@pytest.mark.parametrize("groups,beams,count", [(1, 1, 1), (2, 4, 8), (3, 3, 2), (1, 16, 32), (2, 8, 8)])
def test_vocabularies_of_many_lengths(device, io, vocab, groups, beams, count):
    logits, scores = rows_of(groups, beams, vocab, io, vocab + beams)
    check(device, logits, scores, beams, min(count, beams * vocab))


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("count", [1, 3, 31, 33, 64, 65, 100, 128])
def test_counts(device, io, count):
    """Up to the most; with one beam all of them come from one row, and from one chunk where the row falls."""
    import torch

    logits, scores = rows_of(2, 2, 9000, io, count)
    check(device, logits, scores, 2, count)
    falling = -torch.arange(20000.0)[None].expand(2, -1) / 64
    check(device, falling.to(getattr(torch, io)), [-1.0, -2.0], 1, count)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups,beams", [(64, 8), (5, 64), (130, 1)])
def test_many_rows(device, io, groups, beams):
    logits, scores = rows_of(groups, beams, 9001, io, groups)
    check(device, logits, scores, beams, min(2 * beams, 128))


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 3000, 20000])
def test_equal_logits_and_scores(device, io, vocab):
    import torch

    dtype = getattr(torch, io)
    check(device, torch.zeros((6, vocab), dtype=dtype), [-1.0, -2.0, -1.0, 0.0, 0.0, 0.0], 3, 20)
    few = torch.randint(0, 3, (6, vocab), generator=torch.Generator().manual_seed(1)).to(dtype)
    check(device, few, [-1.0, -1.0, -1.0, 0.0, 0.0, 0.0], 3, 40)
    same = torch.randn((1, vocab), generator=torch.Generator().manual_seed(2)).to(dtype).expand(8, -1).contiguous()
    check(device, same, np.full(8, -3.0), 4, 32)  # four beams of the same row: by their order
    signs = torch.zeros((2, vocab), dtype=dtype)
    signs[:, ::2] = -0.0
    check(device, signs, [0.0, 0.0], 2, 8)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
def test_ended_dead_and_bad_beams(device, io):
    logits, scores = rows_of(8, 4, 3000, io, 3)
    finished = np.zeros(32, bool)
    scores[1:4] = -math.inf  # group 0: the first token of a request
    finished[4:6] = True  # group 1: two have ended
    finished[8:12] = True  # group 2: all have
    scores[12:16] = -math.inf  # group 3: nothing counts
    scores[16], scores[17] = math.nan, math.inf
    logits[20, 17], logits[21, 5], logits[22] = math.nan, math.inf, -math.inf
    finished[24], scores[24] = True, -math.inf  # an ended beam that does not count
    logits[28:31] = math.nan  # rows that nobody looks at
    finished[28], scores[29], scores[30] = True, -math.inf, math.nan
    check(device, logits, scores, 4, 8, finished, 2999)
    check(device, logits, scores, 4, 8, None, 7)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("count", [4, 64, 100])
def test_masked_vocabularies(device, io, count):
    """Logits of -inf: all but a few, all but a stretch, and in places that leave one lane of every wavefront without any."""
    logits, scores = rows_of(6, 2, 20011, io, count)
    logits[0:2, 3:-2] = -math.inf
    logits[2:4, :9000] = -math.inf
    logits[2:4, 9700:] = -math.inf
    import torch

    token = torch.arange(20011)
    for row, width in ((4, 4), (5, 8)):
        logits[row, (token // width) % 64 == 0] = -math.inf
    logits[6, (token // 4) % 4 == 1] = -math.inf
    logits[8, 1:] = -math.inf
    logits[9, :] = -math.inf
    check(device, logits, scores, 2, count)


def test_large_and_small_logits_and_far_scores(device):
    import torch

    logits, _ = rows_of(4, 4, 5000, "float32", 1)
    logits[0:4] *= 1e4
    logits[4:8] *= 1e-6
    logits[8:12] += 3e4
    logits[12:16] *= 1e30
    check(device, logits, [-1e-3, -40.0, 0.0, -1e5, *np.linspace(-1, 0, 4), -1e6, 1e6, 0.0, 5.0, -2.0, -1.0, 0.0, -1e10], 4, 8)
    # Beams whose scores differ by less than float32 holds of them: their order is that of the unrounded ones.
    row = torch.randn((1, 4000), generator=torch.Generator().manual_seed(5)) * 3
    near = torch.cat([row, row + 1.0, row - 3e-7, row * 1.0000002])
    check(device, near, [-50.0, -50.0, -50.0, -50.0], 4, 16)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("count", [8, 100, 128])
def test_plateaus_at_the_last_place(device, io, count):
    """More equal logits than a list holds, of which the first tokens are taken: above them nothing, some, or all but one."""
    import torch

    vocab = 20000
    logits = torch.zeros((6, vocab), dtype=getattr(torch, io))
    gen = torch.Generator().manual_seed(count)
    for row, above in enumerate((0, 3, count // 2, count - 1, count, 5000)):
        at = torch.randperm(vocab, generator=gen)[:above]
        logits[row, at] = 1 + torch.arange(above).to(logits.dtype) / 64 if above < 5000 else 1.0
    logits[2, torch.arange(vocab) % 3 == 0] = -1.0
    for beams in (1, 3, 6):
        check(device, logits, np.zeros(6), beams, count)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [200, 3000, 20000])
def test_many_beams_of_equal_rows(device, io, vocab):
    """64 beams with the same candidates at equal scores: more than a list holds, by beams and then tokens."""
    import torch

    row = torch.randn((1, vocab), generator=torch.Generator().manual_seed(vocab)).to(getattr(torch, io))
    check(device, row.expand(64, -1).contiguous(), np.full(64, -2.0), 64, 128)
    check(device, torch.zeros((64, vocab), dtype=row.dtype), np.zeros(64), 64, 128)
    scores = np.full(64, -1.0)
    scores[5:] = -math.inf  # five of them count
    check(device, torch.zeros((64, vocab), dtype=row.dtype), scores, 64, 128)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
def test_one_beam_far_above_the_others(device, io):
    logits, _ = rows_of(2, 16, 9000, io, 5)
    scores = np.full(32, -1000.0)
    scores[3], scores[16:] = 0.0, -math.inf
    scores[20] = -7.0
    for count in (16, 32, 128):
        check(device, logits, scores, 16, count)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
def test_logits_further_apart_than_exponents(device, io):
    """A thread's first logits tell it little of its others: rising and falling rows, masked beginnings, one high logit anywhere."""
    import torch

    dtype = getattr(torch, io)
    ramp = torch.arange(9000.0)
    logits = torch.stack([ramp, -ramp, ramp * 1e34, -ramp * 1e34, torch.full((9000,), 2e38), torch.full((9000,), -2e38), ramp % 2 * 5e3, ramp % 7 * -3e3]).to(dtype)
    check(device, logits, np.zeros(8), 2, 4, near=True)
    masked = torch.full((4, 9000), -math.inf, dtype=dtype)
    for row, (every, value) in enumerate(((16, 3000.0), (32, -3000.0), (8191, 1e30), (8192, -1e30))):
        masked[row, every - 1 :: every] = value
    check(device, masked, np.zeros(4), 1, 1)
    check(device, masked, np.zeros(4), 2, 3)
    high, _ = rows_of(3, 8, 9000, io, 9)
    for row in range(24):
        high[row, row * 373 + 5] = 4000.0 + row
    check(device, high, np.linspace(0, -1, 24), 8, 8)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("level", [-600.0, -655.0, -690.0, -700.0, -709.0, -709.8, -711.0, -1000.0, -2110.0, -2120.0, -2130.0, -3549.0, -4970.0])
def test_rows_far_below_zero(device, io, level):
    """A thread without a finite logit (behind the vocabulary's end, or masked) adds nothing, wherever the others lie."""
    import torch

    dtype = getattr(torch, io)
    for vocab in (200, 1000, 2049, 9001):
        logits, scores = rows_of(2, 4, vocab, "float32", vocab)
        check(device, (logits + level).to(dtype), scores, 4, 8)
        masked = torch.full(logits.shape, -math.inf)
        for row in range(8):  # some tokens of the row, or a stretch
            at = torch.arange(vocab) % 37 == row if row % 2 else (torch.arange(vocab) >= 20 * row) & (torch.arange(vocab) < 20 * row + 40)
            masked[row, at] = logits[row, at] + level
        check(device, masked.to(dtype), scores, 4, 8)
    # Ordinary rows, of which one chunk or the last numbers hold such logits alone, with and without masked ones between.
    for vocab in (2060, 9001):
        logits, scores = rows_of(2, 4, vocab, "float32", vocab)
        logits[::2, 2048:] += level
        logits[1::2, -12:] += level
        logits[2:4, 2050::3] = -math.inf
        check(device, logits.to(dtype), scores, 4, 8)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [5, 2048, 9000])
def test_one_bad_logit_anywhere(device, io, vocab):
    logits, scores = rows_of(3, 8, vocab, io, vocab)
    for row in range(0, 24, 2):
        logits[row, row * 7919 % vocab] = (math.nan, math.inf)[row // 2 % 2]
    check(device, logits, scores, 8, 8)


def test_rows_with_strides_and_given_buffers(device):
    import torch

    from paged_kv_serving_amd import ops

    wide = torch.randn((6, 5009))
    for io in (torch.float32, torch.bfloat16):
        base = wide.to(io)
        for view in (base[:, :4999], base[:, 1:5000], base[::2][:3, 3:]):
            rows = view.shape[0]
            scores = -np.arange(rows)
            want = check(device, view.contiguous(), scores, 3, 6)
            held = base.to(device)
            there = torch.as_strided(held, view.shape, view.stride(), view.storage_offset())
            got = ops.beam_select(there, torch.as_tensor(scores, dtype=torch.float32).to(device), num_beams=3, count=6)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        turned = base[:, :1000].t().contiguous().to(device).t()  # columns next to each other
        got = ops.beam_select(turned, torch.zeros(6, device=device), num_beams=2, count=4)
        for a, b in zip(got, check(device, base[:, :1000].contiguous(), np.zeros(6), 2, 4)):
            assert torch.equal(a, b)
    need = ops.beam_workspace_bytes(2, 3, 5009, 6)
    workspace = torch.full((need + 16,), 255, dtype=torch.uint8, device=device)[:need]
    out = ops.BeamChoice(torch.zeros((2, 6), device=device), *(torch.zeros((2, 6), dtype=torch.int32, device=device) for _ in range(2)))
    assert check(device, wide, np.zeros(6), 3, 6, out=out, workspace=workspace) is out
    assert select(device, wide[:0], np.zeros(0), 3, 6).scores.shape == (0, 6)


def test_a_row_does_not_depend_on_the_batch(device):
    import torch

    logits, scores = rows_of(80, 4, 9000, "float32", 2)
    whole = select(device, logits, scores, 4, 8)
    alone = [select(device, logits[4 * g : 4 * g + 4], scores[4 * g : 4 * g + 4], 4, 8) for g in range(0, 80, 13)]
    for g, one in zip(range(0, 80, 13), alone):
        for a, b in zip(whole, one):
            assert torch.equal(a[g], b[0])
    again = select(device, logits, scores, 4, 8)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))


def test_two_streams_at_once_and_a_replayed_graph(device):
    import torch

    from paged_kv_serving_amd import ops

    both = []
    for seed, (groups, beams, vocab, io) in enumerate(((3, 4, 30000, "float32"), (40, 8, 9001, "bfloat16"))):
        logits, scores = rows_of(groups, beams, vocab, io, seed)
        both.append((logits.to(device), torch.as_tensor(scores, dtype=torch.float32).to(device), beams))
    want = [ops.beam_select(x, s, num_beams=b, count=2 * b) for x, s, b in both]
    streams = [torch.cuda.Stream(device) for _ in both]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (x, s, b) in enumerate(both):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.beam_select(x, s, num_beams=b, count=2 * b))
    torch.cuda.synchronize()
    for results, expected in zip(got, want):
        for result in results:
            assert all(torch.equal(a, e) for a, e in zip(result, expected))
    x, s, b = both[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.beam_select(x, s, num_beams=b, count=2 * b)
    for step in range(4):
        x.copy_(x.roll(step, 1) * (1 + step))
        s.sub_(float(step))
        graph.replay()
        eager = ops.beam_select(x, s, num_beams=b, count=2 * b)
        assert all(torch.equal(a, e) for a, e in zip(held, eager))


@pytest.mark.parametrize("groups,vocab", [(1, 700), (300, 700), (40, 9001)])
def test_scores_updated_in_place(device, groups, vocab):
    """The best scores over the scores, where there are as many; in other parts of their memory they are refused."""
    import torch

    from paged_kv_serving_amd import ops

    beams = 4
    logits, scores = rows_of(groups, beams, vocab, "float32", groups)
    logits, before = logits.to(device), torch.as_tensor(scores, dtype=torch.float32).to(device)
    held = before.clone()
    for _ in range(3):
        want = ops.beam_select(logits, before, num_beams=beams)
        out = ops.BeamChoice(held.view(groups, beams), torch.empty_like(want.beams), torch.empty_like(want.tokens))
        got = ops.beam_select(logits, held, num_beams=beams, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and got.scores.data_ptr() == held.data_ptr()
        before = want.scores.view(-1)
    room = torch.zeros(5 * groups * beams, device=device)
    rows = groups * beams
    for count, first in ((2 * beams, 0), (2 * beams, 1), (beams, 1), (beams, rows - 1), (2, 0)):
        for a, b in ((0, first), (2 * rows, 2 * rows - first)):  # where the scores begin, and the best ones
            out = ops.BeamChoice(room[b : b + groups * count].view(groups, count), *(torch.empty((groups, count), dtype=torch.int32, device=device) for _ in range(2)))
            with pytest.raises(ValueError, match="memory"):
                ops.beam_select(logits, room[a : a + rows], num_beams=beams, count=count, out=out)


def test_select_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    good = dict(logits=torch.zeros((6, 50), device=device), scores=torch.zeros(6, device=device), num_beams=3)
    assert ops.beam_select(**good).scores.shape == (2, 3)
    out = ops.beam_select(**good)
    bad = [
        {"logits": good["logits"].half()}, {"logits": good["logits"][0]}, {"logits": torch.zeros((6, 0), device=device)}, {"num_beams": 4}, {"num_beams": 0}, {"count": 0},
        {"count": 151}, {"count": 129}, {"scores": torch.zeros(5, device=device)}, {"scores": torch.zeros(6, device=device).double()}, {"scores": torch.zeros(6)},
        {"scores": torch.zeros(12, device=device)[::2]}, {"finished": torch.zeros(6, device=device)}, {"finished": torch.zeros(5, dtype=torch.bool, device=device)},
        {"end_token": -1}, {"end_token": 1 << 31}, {"out": out._replace(tokens=out.scores)}, {"out": ops.BeamChoice(*(x[:1] for x in out))},
        {"workspace": torch.zeros(2, device=device)}, {"workspace": torch.zeros(10**6)}, {"logits": torch.zeros((130, 9), device=device), "scores": torch.zeros(130, device=device), "num_beams": 65},
    ]  # fmt: skip
    for change in bad:
        with pytest.raises(ValueError):
            ops.beam_select(**{**good, **change})
    for sizes in ((-1, 2, 10, 1), (1, 65, 10, 1), (1, 2, 0, 1), (1, 2, 1 << 26, 1), (1, 2, 10, 129), (1 << 20, 2, 10, 1)):
        with pytest.raises(ValueError):
            ops.beam_workspace_bytes(*sizes)


# --- reordering ---------------------------------------------------------------------------------


def beams_of(groups, beams, block, width, layers, shapes, contexts, seed):
    """Tables whose rows share a few leading blocks and have their last ones to themselves, and states of random bytes."""
    import torch

    rng = np.random.default_rng(seed)
    used = -(-contexts // block)
    shared = np.minimum(rng.integers(0, 4, groups), contexts // block)
    blocks = int((shared + beams * (used - shared)).sum()) + 3
    ids = rng.permutation(blocks)
    tables, at = rng.integers(-5, blocks + 5, (groups, beams, width)), 0  # behind a row's blocks: anything
    for g in range(groups):
        tables[g, :, : shared[g]] = ids[at : at + shared[g]]
        at += shared[g]
        for b in range(beams):
            n = used[g] - shared[g]
            tables[g, b, shared[g] : used[g]] = ids[at : at + n]
            at += n
    gen = torch.Generator().manual_seed(seed)
    states = [torch.randint(0, 256, (n, blocks, size), generator=gen, dtype=torch.uint8) for n, size in zip(layers, shapes)]
    return tables.astype(np.int32), states


def check_reorder(device, tables, parents, contexts, states, block, given=None):
    import torch

    from paged_kv_serving_amd import ops

    groups, beams, width = tables.shape
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)  # noqa: E731
    held = [s.to(device) for s in states] if given is None else given
    out = ops.beam_reorder(put(tables).view(groups * beams, width), put(parents), put(contexts), held, block_size=block)
    want, copies = np.zeros_like(tables), []
    for g in range(groups):
        want[g], more = reorder_group(tables[g], parents[g].tolist(), int(contexts[g]), block)
        copies += more
    np.testing.assert_array_equal(out.cpu().numpy().reshape(tables.shape), want)
    for state, after in zip(states, held):
        expected = state.clone()
        for source, target in copies:
            expected[:, target] = state[:, source]
        assert torch.equal(after.cpu().view(torch.uint8).reshape(expected.shape), expected)
    return copies


@pytest.mark.parametrize("block", [1, 4, 16])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 2), (3, 4), (7, 5), (2, 64), (40, 8)])
def test_random_parents(device, groups, beams, block):
    rng = np.random.default_rng(groups + beams + block)
    for seed in range(3):
        contexts = rng.integers(1, 9 * block + 1, groups)
        tables, states = beams_of(groups, beams, block, 12, (3, 3, 1), (64, 4100, 12), contexts, seed)
        spread = rng.integers(0, beams, (groups, beams)) if seed else np.minimum(rng.geometric(0.4, (groups, beams)) - 1, beams - 1)
        check_reorder(device, tables, spread, contexts, states, block)


def test_parents_of_every_kind(device):
    """All of one row, every row its own, rows exchanged, the last row only, parents outside the group."""
    parents = np.asarray([[0, 0, 0, 0], [0, 1, 2, 3], [1, 0, 3, 2], [3, 3, 3, 3], [2, 2, 0, 0], [-1, 4, 0, 2**31 - 1], [3, 2, 1, 0], [1, 1, 1, 2]])
    contexts = np.asarray([7, 7, 9, 10, 1, 6, 3, 8])
    tables, states = beams_of(8, 4, 4, 5, (2, 2), (100, 7), contexts, 1)
    copies = check_reorder(device, tables, parents, contexts, states, 4)
    assert len(copies) == 3 + 0 + 0 + 3 + 2 + 1 + 0 + 0  # the last group's context ends with a full block


@pytest.mark.parametrize("size", [1, 3, 4, 16, 20, 48, 4096, 5000, 16384, 70000])
def test_blocks_of_many_sizes_and_alignments(device, size):
    import torch

    contexts = np.asarray([9, 5])
    tables, states = beams_of(2, 3, 4, 4, (2,), (size,), contexts, size)
    parents = np.asarray([[1, 1, 1], [2, 0, 2]])
    assert len(check_reorder(device, tables, parents, contexts, states, 4)) == 3
    for shift in (1, 4):  # a state that begins anywhere
        flat = torch.zeros(states[0].numel() + 32, dtype=torch.uint8, device=device)
        view = flat[shift : shift + states[0].numel()].view(states[0].shape)
        view.copy_(states[0])
        check_reorder(device, tables, parents, contexts, states, 4, given=[view])
        assert not flat[:shift].any() and not flat[shift + states[0].numel() :].any()


@pytest.mark.parametrize("sizes", [(64, 4, 16, 1, 1000, 48, 7, 2048), (3, 5), (256, 257), (4096, 4096, 4, 4), (4096, 4112, 4, 4)])
def test_states_of_different_sizes(device, sizes):
    """Blocks that a wavefront moves by itself, and one byte more than those."""
    rng = np.random.default_rng(3)
    contexts = rng.integers(1, 40, 9)
    tables, states = beams_of(9, 4, 8, 12, tuple(range(1, len(sizes) + 1)), sizes, contexts, 3)
    check_reorder(device, tables, rng.integers(0, 4, (9, 4)), contexts, states, 8)


def test_a_cache_of_codes_and_scales(device):
    """An 8-bit cache: codes and scales of both kinds, moved in one call."""
    import torch

    contexts = np.asarray([21, 40, 33])
    block, kv_heads, dim, layers = 16, 2, 32, 3
    tables, states = beams_of(3, 4, block, 4, (layers,) * 4, (block * kv_heads * dim,) * 2 + (4 * kv_heads,) * 2, contexts, 3)
    blocks = states[0].shape[1]
    held = [s.to(device) for s in states]
    given = [
        *(h.view(layers, blocks, block, kv_heads, dim).view(torch.float8_e4m3fn) for h in held[:2]),
        *(h.contiguous().view(torch.float32).view(layers, blocks, kv_heads) for h in held[2:]),
    ]  # fmt: skip
    parents = np.asarray([[0, 0, 0, 1], [3, 3, 1, 1], [2, 2, 2, 2]])
    check_reorder(device, tables, parents, contexts, states, block, given=given)


def test_blocks_and_contexts_outside(device):
    """Tables that name blocks outside the pool, contexts outside the table: no state is touched there."""
    contexts = np.asarray([6, 100, -4, 0])
    tables, states = beams_of(4, 3, 4, 3, (2,), (36,), np.asarray([6, 12, 1, 1]), 5)
    tables[0, 0, 1], tables[0, 2, 1] = -1, 10**6
    parents = np.asarray([[0, 0, 1], [1, 1, 1], [2, 2, 2], [0, 0, 0]])
    import torch

    from paged_kv_serving_amd import ops

    held = [s.to(device) for s in states]
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)  # noqa: E731
    out = ops.beam_reorder(put(tables).view(12, 3), put(parents), put(contexts), held, block_size=4)
    want = np.stack([reorder_group(tables[g], parents[g].tolist(), int(contexts[g]), 4)[0] for g in range(4)])
    np.testing.assert_array_equal(out.cpu().numpy().reshape(tables.shape), want)
    assert torch.equal(held[0].cpu(), states[0])


def test_states_past_32_bit_offsets(device):
    import torch

    contexts = np.asarray([6])
    tables, _ = beams_of(1, 2, 4, 3, (1,), (4,), contexts, 1)
    from paged_kv_serving_amd import ops

    size, blocks, layers = 1 << 20, 1100, 4
    state = torch.zeros((layers, blocks, size), dtype=torch.uint8, device=device)
    tables = np.asarray([[[5, blocks - 1, 0], [5, blocks - 2, 0]]], np.int32)
    state[:, blocks - 2] = torch.arange(layers, dtype=torch.uint8, device=device)[:, None] + 1
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)  # noqa: E731
    ops.beam_reorder(put(tables).view(2, 3), put([[1, 1]]), put(contexts), [state], block_size=4)
    assert torch.equal(state[:, blocks - 1], state[:, blocks - 2]) and state[:, blocks - 1].any(1).all() and not state[:, : blocks - 2].any()


def test_new_tables_in_the_memory_of_the_old_ones_are_refused(device):
    import torch

    from paged_kv_serving_amd import ops

    both = torch.arange(48, dtype=torch.int32, device=device).view(12, 4)
    parents, contexts = torch.zeros((2, 3), dtype=torch.int32, device=device), torch.tensor([5, 9], dtype=torch.int32, device=device)
    for first in range(6):
        there = both[first : first + 6]
        for old, new in ((both[:6], there), (there, both[:6])):
            with pytest.raises(ValueError, match="share memory"):
                ops.beam_reorder(old, parents, contexts, [], block_size=4, out=new)
    want = ops.beam_reorder(both[:6].clone(), parents, contexts, [], block_size=4)
    assert torch.equal(ops.beam_reorder(both[:6], parents, contexts, [], block_size=4, out=both[6:]), want)
    narrow = both.view(-1)[:0].view(6, 0)
    assert ops.beam_reorder(narrow, parents, contexts, [], block_size=4, out=narrow).shape == (6, 0)


def test_reorder_without_states_and_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
    good = dict(block_tables=i32(6, 4), parents=i32(2, 3), context_lens=i32(2), states=[torch.zeros((2, 5, 8), device=device)], block_size=4)
    assert ops.beam_reorder(**good).shape == (6, 4)
    assert ops.beam_reorder(**{**good, "states": []}).shape == (6, 4)
    out = i32(6, 4)
    assert ops.beam_reorder(**good, out=out) is out
    assert ops.beam_reorder(i32(0, 4), i32(0, 3), i32(0), [], block_size=4).shape == (0, 4)
    bad = [
        {"block_tables": i32(5, 4)}, {"block_tables": i32(6, 4).long()}, {"block_tables": i32(4, 6).t()}, {"parents": i32(6)}, {"parents": i32(2, 3).long()},
        {"parents": i32(3, 2).t()}, {"context_lens": i32(3)}, {"context_lens": i32(2).long()}, {"block_size": 0}, {"states": [torch.zeros(5, device=device)]},
        {"states": [torch.zeros((2, 5, 8), device=device), torch.zeros((2, 6, 8), device=device)]}, {"states": [torch.zeros((5, 2, 8), device=device).transpose(0, 1)]},
        {"states": [torch.zeros((1, 5, 4), device=device)] * 9}, {"states": [torch.zeros((2, 5, 8))]}, {"out": i32(6, 3)}, {"out": good["block_tables"]},
        {"block_tables": i32(130, 4), "parents": i32(2, 65)},
    ]  # fmt: skip
    for change in bad:
        with pytest.raises(ValueError):
            ops.beam_reorder(**{**good, **change})
