"""Beam search over an 8-bit paged cache, as the operators are used together: step_metadata, rope_append_axes,
append_kv_e4m3, paged_attention_e4m3, beam_select and beam_reorder, eager and as one replayed graph. Every beam's cache is compared
with one that was filled with its tokens alone."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import e4m3
from oracle.beam import select_group
from oracle.window import window_attention
from paged_kv_serving_amd import ops

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, HALF, BLOCK, VOCAB = 8, 2, 64, 32, 8, 300
PROMPTS, BEAMS, STEPS = (5, 16, 27), 3, 13
END = 17


class Search:
    """One attention layer over an 8-bit cache, whose projections are rows of a table by token id."""

    def __init__(self, device, dtype) -> None:
        gen = torch.Generator().manual_seed(7)
        rows = lambda heads: torch.randn((VOCAB, heads, DIM), generator=gen).to(dtype).to(device)  # noqa: E731
        self.q, self.k, self.v = rows(HEADS), rows(KV_HEADS), rows(KV_HEADS)
        self.head = (torch.randn((HEADS * DIM, VOCAB), generator=gen) / 8).to(device)
        angles = torch.arange(100)[:, None] / 1000.0 ** (torch.arange(HALF) / HALF)
        self.cos, self.sin = torch.cos(angles).float().to(device), torch.sin(angles).float().to(device)
        self.device, self.groups, self.rows = device, len(PROMPTS), len(PROMPTS) * BEAMS
        blocks = 100
        self.pools = [torch.zeros((1, blocks, BLOCK, KV_HEADS, DIM), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        self.scales = [torch.zeros((1, blocks, KV_HEADS), device=device) for _ in range(2)]
        ids = torch.from_numpy(np.random.default_rng(3).permutation(blocks).astype(np.int32)).to(device)
        # Every row but a group's first has a last block of its own, for the prompt's part of one.
        self.tables = torch.zeros((self.rows, 8), dtype=torch.int32, device=device)
        for g, prompt in enumerate(PROMPTS):
            for b in range(1, BEAMS):
                self.tables[g * BEAMS + b, prompt // BLOCK] = ids[g * BEAMS + b]
        self.free = ids[self.rows :].contiguous()
        i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        first = [p if b == 0 else 0 for p in PROMPTS for b in range(BEAMS)]
        self.query, self.contexts, self.group_contexts, self.next_free = i32(first), i32(first), i32(PROMPTS), i32([0])
        self.scores = torch.as_tensor([0.0 if b == 0 else -np.inf for _ in PROMPTS for b in range(BEAMS)], dtype=torch.float32, device=device)
        self.finished = torch.zeros(self.rows, dtype=torch.bool, device=device)
        self.last = torch.as_tensor(np.cumsum(first) - 1, device=device).clamp(min=0)  # rows whose logits count
        self.base = torch.arange(self.rows, device=device) // BEAMS * BEAMS

    def step(self, tokens, num_rows: int, most: int):
        """One step of all rows: its attention, logits and choice; tables, scores and ended beams move on."""
        m = ops.step_metadata(self.query, self.contexts, self.tables, self.free, self.next_free, block_size=BLOCK, num_rows=num_rows)
        rotated = torch.empty((2, num_rows, 1, KV_HEADS, DIM), dtype=self.k.dtype, device=self.device)  # a pool of a slot for each row
        slots = torch.arange(num_rows, device=self.device)
        queries = ops.rope_append_axes(rotated[0], rotated[1], self.q[tokens], self.k[tokens], self.v[tokens], m.positions, self.cos, self.sin, slots)
        ops.append_kv_e4m3(self.pools[0][0], self.pools[1][0], self.scales[0][0], self.scales[1][0], rotated[0][:, 0], rotated[1][:, 0], m.slot_mapping)
        out = ops.paged_attention_e4m3(queries, m.query_positions, m.query_seq, self.pools[0][0], self.pools[1][0], self.scales[0][0], self.scales[1][0],
                                       self.tables, m.context_lens, DIM**-0.5, max_context_len=64, max_query_len=most)  # fmt: skip
        logits = out.flatten(1).float()[self.last] @ self.head
        best = ops.beam_select(logits, self.scores, num_beams=BEAMS, finished=self.finished, end_token=END)
        tables = ops.beam_reorder(self.tables, best.beams, self.group_contexts, [*self.pools, *self.scales], block_size=BLOCK)
        ended = self.finished[self.base + best.beams.flatten().long()] | (best.tokens.flatten() == END)
        self.tables.copy_(tables)
        self.next_free.copy_(m.next_free)
        self.scores.copy_(best.scores.flatten())
        self.finished.copy_(ended)
        return queries, out, logits, best, m

    def grow(self):
        """From a step to the next: a token more for every row."""
        self.contexts.add_(1)
        self.group_contexts.add_(1)


def decode_inputs(s):
    s.query.fill_(1)
    for g, p in enumerate(PROMPTS):
        s.contexts[g * BEAMS : (g + 1) * BEAMS] = p
    s.last = torch.arange(s.rows, device=s.device)


def cache_of(s, history, prompt):
    """Codes and scales of a cache that was filled with one beam's tokens: its prompt, then one after the other."""
    blocks = -(-len(history) // BLOCK)
    tokens = torch.as_tensor(history, device=s.device)
    k, v = torch.zeros((2, len(history), 1, KV_HEADS, DIM), dtype=s.k.dtype, device=s.device)
    ops.rope_append_axes(k, v, s.q[tokens], s.k[tokens], s.v[tokens], torch.arange(len(history), device=s.device), s.cos, s.sin,
                         torch.arange(len(history), device=s.device))  # fmt: skip
    out = []
    for new in (k, v):
        new = new[:, 0].float().cpu().numpy()
        codes, scales = np.zeros((blocks, BLOCK, KV_HEADS, DIM)), np.zeros((blocks, KV_HEADS))
        e4m3.append(codes, scales, new[:prompt], np.arange(prompt))
        for t in range(prompt, len(history)):
            e4m3.append(codes, scales, new[t : t + 1], [t])
        out.append((codes, scales))
    return out


def check_caches(s, histories):
    for row, history in enumerate(histories):
        used = -(-len(history) // BLOCK)
        ids = s.tables[row, :used].long()
        for pool, scale, (codes, scales) in zip(s.pools, s.scales, cache_of(s, history, PROMPTS[row // BEAMS])):
            there = pool[0].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float().cpu().numpy()
            np.testing.assert_array_equal(there.reshape(-1, KV_HEADS, DIM)[: len(history)], codes.reshape(-1, KV_HEADS, DIM)[: len(history)])
            np.testing.assert_array_equal(scale[0][ids].cpu().numpy(), scales)


def check_choice(logits, scores, finished, best):
    rows = logits.cpu().numpy()
    for g in range(len(PROMPTS)):
        at = slice(g * BEAMS, (g + 1) * BEAMS)
        want = select_group(rows[at], scores[at], BEAMS, finished[at], END)
        assert list(zip(best.beams[g].tolist(), best.tokens[g].tolist())) == [(b, t) for _, b, t in want]
        assert np.allclose(best.scores[g].cpu().numpy(), [x for x, _, _ in want], rtol=2.0**-22, atol=0)


def prompts():
    rng = np.random.default_rng(5)
    return [rng.integers(0, VOCAB, p).tolist() for p in PROMPTS]


def start(s):
    """The prompts' step; the histories of all rows after it and the tokens that follow."""
    texts = prompts()
    tokens = torch.as_tensor(sum(texts, []), device=s.device)
    queries, out, logits, best, m = s.step(tokens, int(sum(PROMPTS)), max(PROMPTS))
    assert m.query_starts.tolist()[-1] == sum(PROMPTS)
    return texts, best, logits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_search_step_by_step(device, dtype):
    s = Search(device, dtype)
    scores, finished = s.scores.cpu().numpy(), s.finished.cpu().numpy()
    texts, best, logits = start(s)
    check_choice(logits, scores, finished, best)
    histories = [texts[row // BEAMS] for row in range(s.rows)]
    following = best.tokens.flatten().tolist()
    decode_inputs(s)
    for step in range(STEPS):
        check_caches(s, histories)
        s.grow()
        scores, finished = s.scores.cpu().numpy(), s.finished.cpu().numpy()
        before = s.tables.clone()
        queries, out, logits, best, m = s.step(torch.as_tensor(following, device=device), s.rows, 1)
        histories = [h + [t] for h, t in zip(histories, following)]
        # The attention of every row over its own beam's cache.
        for row, history in enumerate(histories):
            (k, ks), (v, vs) = cache_of(s, history, PROMPTS[row // BEAMS])
            want, size = window_attention(queries[row : row + 1].float().cpu().numpy(), [len(history) - 1], [0], e4m3.values(k, ks), e4m3.values(v, vs),
                                       np.arange(k.shape[0])[None], [len(history)], DIM**-0.5, 1 << 20, 0)  # fmt: skip
            # A score is off by (dim + 8) 2^-24 of scale * sum |q k| at most, which moves a weight by twice as much; sums of n
            # terms by n 2^-24; a bfloat16 row's weights are rounded to 2^-17 at most and its result once.
            most, scores_off = np.abs(e4m3.values(v, vs)).max(), (DIM + 8) * 2.0**-24 * size[0][:, None]
            bound = most * (2 * np.expm1(2 * scores_off) + (len(history) + 16) * 2.0**-24)
            if dtype == torch.bfloat16:
                bound = bound + most * 2.0**-16 + np.abs(want[0]) * 2.0**-8
            assert (np.abs(out[row].float().cpu().numpy() - want[0]) <= bound).all()
        check_choice(logits, scores, finished, best)
        parents = (s.base + best.beams.flatten().long()).tolist()
        histories = [histories[p] for p in parents]
        following = best.tokens.flatten().tolist()
        assert before.shape == s.tables.shape
    check_caches(s, histories)
    assert len({tuple(h) for h in histories}) > s.groups  # beams did part


def test_the_same_search_as_a_replayed_graph(device):
    eager, captured = Search(device, torch.bfloat16), Search(device, torch.bfloat16)
    choices = []
    for s in (eager, captured):
        _, best, _ = start(s)
        decode_inputs(s)
        s.tokens = best.tokens.flatten().long().clone()
    for _ in range(STEPS):
        eager.grow()
        _, _, _, best, _ = eager.step(eager.tokens, eager.rows, 1)
        eager.tokens.copy_(best.tokens.flatten())
        choices.append([x.clone() for x in best])

    def run():
        captured.grow()
        best = captured.step(captured.tokens, captured.rows, 1)[3]
        captured.tokens.copy_(best.tokens.flatten())
        return best

    # A step run once beforehand, on copies of what it changes, so that capturing meets nothing for the first time.
    kept = [x.clone() for x in (captured.tables, captured.next_free, captured.scores, captured.finished, captured.contexts, captured.group_contexts, captured.tokens,
                                *(p.view(torch.uint8) for p in captured.pools), *captured.scales)]  # fmt: skip
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        best = run()
    for x, y in zip((captured.tables, captured.next_free, captured.scores, captured.finished, captured.contexts, captured.group_contexts, captured.tokens,
                     *(p.view(torch.uint8) for p in captured.pools), *captured.scales), kept):  # fmt: skip
        x.copy_(y)
    for want in choices:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(best, want):
            assert torch.equal(a, b)
    assert torch.equal(captured.tables, eager.tables)
    for a, b in zip((*captured.pools, *captured.scales), (*eager.pools, *eager.scales)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
