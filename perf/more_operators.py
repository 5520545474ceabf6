"""The operators of serving from an 8-bit cache and of beam search, as they are measured.

Five kinds of pass, each one call of a serving step:

    append   ops.append_kv_e4m3: new keys and values to a paged cache of 8-bit floats (e4m3) with a power of two
             as the scale of each block of tokens and head
    attend   ops.paged_attention_e4m3: attention over that cache, decode rows and prompt chunks in one ragged batch
    step     ops.step_metadata: rows, positions and slots of a step from its requests' lengths, and their block
             tables extended from a list of free blocks
    select   ops.beam_select: the best continuations of each group of beams over the whole vocabulary
    reorder  ops.beam_reorder: block tables and the last, partly filled blocks of beams moved to the beams that go on

Sizes are those of this repository's configurations, benchmark and tests (blocks of 16, chunks of 512, contexts up to
32,768, vocabularies of 50,257 and 128,256, heads of 64 and 128) and generic ones between them.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0  # of e4m3
LOW_EXPONENT = -100  # of a scale


def listed() -> list[dict]:
    return [
        # A decode step's append of a full batch: a token each. Latency.
        {"name": "append_64_bf16", "kind": "append", "seqs": 64, "low": 500, "high": 2000, "chunks": 0, "chunk": 0, "kv_heads": 8, "dim": 128, "io": "bf16", "block": 16},
        # The tokens of a full step of prompt chunks beside decode rows, float32 activations.
        {"name": "append_8x512_120_f32", "kind": "append", "seqs": 120, "low": 1, "high": 300, "chunks": 8, "chunk": 512, "kv_heads": 32, "dim": 128, "io": "f32", "block": 16},
        # One interactive sequence. Latency.
        {"name": "attend_decode_1", "kind": "attend", "seqs": 1, "low": 3900, "high": 3900, "chunks": 0, "chunk": 0, "offset": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0, "io": "bf16", "block": 16},
        # A decode step of 64 sequences, short and long ones.
        {"name": "attend_decode_64_bf16", "kind": "attend", "seqs": 64, "low": 2048, "high": 32768, "chunks": 0, "chunk": 0, "offset": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 0, "sinks": 0, "io": "bf16", "block": 16},
        # The prompt chunks of a full step, grouped heads.
        {"name": "attend_prefill_8x512_bf16", "kind": "attend", "seqs": 0, "low": 0, "high": 0, "chunks": 8, "chunk": 512, "offset": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 0, "sinks": 0, "io": "bf16", "block": 16},
        # Odd-sized chunks beside decode rows under a window, float32 activations.
        {"name": "attend_mixed_2x301_24_f32", "kind": "attend", "seqs": 24, "low": 100, "high": 4000, "chunks": 2, "chunk": 301, "offset": 700, "heads": 16, "kv_heads": 16,
         "dim": 64, "window": 1000, "sinks": 5, "io": "f32", "block": 16},
        # A decode step's metadata: a row each, tables for long contexts. Latency.
        {"name": "step_64", "kind": "step", "seqs": 64, "chunks": 0, "chunk": 0, "high": 32000, "block": 16, "width": 2048, "rows": 64},
        # A full step of prompt chunks beside decode rows, padded to a captured step's rows.
        {"name": "step_32x512_250", "kind": "step", "seqs": 250, "chunks": 32, "chunk": 512, "high": 16000, "block": 16, "width": 2048, "rows": 16896},
        # One request's beams. Latency.
        {"name": "select_1x4_32000", "kind": "select", "groups": 1, "beams": 4, "count": 8, "vocab": 32000, "io": "f32"},
        # A batch of requests, a large vocabulary.
        {"name": "select_32x8_128256", "kind": "select", "groups": 32, "beams": 8, "count": 16, "vocab": 128256, "io": "f32"},
        # One request's beams, 16-bit cache of a few layers. Latency.
        {"name": "reorder_1x4", "kind": "reorder", "groups": 1, "beams": 4, "layers": 4, "kv_heads": 8, "dim": 64, "cache": "bf16", "block": 16, "width": 64, "context": 500},
        # A batch of requests over the 8-bit cache of all layers.
        {"name": "reorder_32x8_e4m3", "kind": "reorder", "groups": 32, "beams": 8, "layers": 32, "kv_heads": 8, "dim": 128, "cache": "e4m3", "block": 16, "width": 128, "context": 1003},
    ]  # fmt: skip


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    """One more case of the ranges above; none costs more than the largest listed ones."""
    kind = rng.choices(["append", "attend", "step", "select", "reorder"], [3, 6, 2, 3, 2])[0]
    block = rng.choice([1, 7, 16, 16, 16, 32, 64])
    if kind == "step":
        seqs, chunks, chunk = _log(rng, 1, 512), rng.choice([0, 0, rng.randint(1, 32)]), _log(rng, 2, 512)
        high = _log(rng, 16, 32000)
        rows = seqs + chunks * chunk + rng.choice([0, 0, rng.randint(1, 64)])
        return {"kind": kind, "seqs": seqs, "chunks": chunks, "chunk": chunk if chunks else 0, "high": high, "block": block,
                "width": -(-(high + 512) // block) + rng.randint(0, 9), "rows": rows}  # fmt: skip
    if kind == "select":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 8, 16]), _log(rng, 200, 128256)
        groups = min(_log(rng, 1, 64), max(1, 256 * 128256 // (beams * vocab)))
        return {"kind": kind, "groups": groups, "beams": beams, "count": rng.choice([beams, 2 * beams]), "vocab": vocab, "io": rng.choice(["f32", "f32", "bf16"])}
    kv_heads, group = rng.choice([(1, 8), (2, 4), (2, 7), (4, 4), (4, 8), (8, 1), (8, 4), (16, 1), (8, 2), (1, 16)])
    dim = rng.choice([32, 64, 64, 128, 128, 128, 256]) if kv_heads * group <= 16 else rng.choice([32, 64, 128])
    if kind == "reorder":
        context, layers = _log(rng, 1, 4000), rng.randint(1, 32)
        beams, groups = rng.choice([2, 3, 4, 5, 8, 8, 16]), _log(rng, 1, 32)
        cache = rng.choice(["e4m3", "e4m3", "bf16", "f32"])
        most = 1_000_000_000 // (kv_heads * dim * (context + 3 * beams * block) * {"e4m3": 1, "bf16": 2, "f32": 4}[cache])  # of layers, for one group
        layers = max(1, min(layers, most))
        groups = max(1, min(groups, most // layers))
        return {"kind": kind, "groups": groups, "beams": beams, "layers": layers, "kv_heads": kv_heads, "dim": dim, "cache": cache, "block": block,
                "width": -(-context // block) + rng.randint(0, 30), "context": context}  # fmt: skip
    io = rng.choice(["bf16", "bf16", "f32"])
    mode = rng.choice(["decode", "decode", "prefill", "mixed"])
    if kind == "append":
        seqs = 0 if mode == "prefill" else _log(rng, 1, 256)
        chunks, chunk = (0, 0) if mode == "decode" else (rng.randint(1, 8), _log(rng, 2, 512))
        return {"kind": kind, "seqs": seqs, "low": 1, "high": _log(rng, 2, 1000), "chunks": chunks, "chunk": chunk, "kv_heads": kv_heads, "dim": dim, "io": io, "block": block}
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 16, 4096), rng.choice([0, 1, 4, 16]))])
    high = _log(rng, 16, 32768)
    seqs = 0 if mode == "prefill" else max(1, min(_log(rng, 1, 64), 1_000_000_000 // (2 * kv_heads * dim * high)))
    chunks = 0 if mode == "decode" else rng.randint(1, 8 if mode == "prefill" else 2)
    chunk = 0 if mode == "decode" else _log(rng, 2, 512)
    offset = 0 if mode == "decode" else _log(rng, 1, 4096) - 1
    while chunks * chunk * (offset + chunk) > 6_000_000:  # (row, key) pairs of the largest listed case
        chunk = chunk * 3 // 4
    if mode == "mixed":  # the plain form pads every sequence to the longest run of rows
        high = min(high, 4000)
        seqs = max(1, min(seqs, 600_000_000 // (kv_heads * group * chunk * max(high, offset + chunk))))
    return {"kind": kind, "seqs": seqs, "low": max(1, int(high * rng.uniform(0.1, 1.0))) if seqs else 0, "high": high if seqs else 0, "chunks": chunks, "chunk": chunk,
            "offset": offset, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "io": io, "block": block}  # fmt: skip


# --- inputs ----------------------------------------------------------------------------------


def _normal(gen: torch.Generator, shape, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _device(array, dtype) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(array)).to(dtype).cuda()


def _codes(gen: torch.Generator, shape) -> torch.Tensor:
    """Codes of a normal distribution whose largest values use the format's range."""
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16) * 110).clamp_(-LARGEST, LARGEST).to(E4M3)


def _scales(gen: torch.Generator, shape, low: int, high: int) -> torch.Tensor:
    return torch.exp2(torch.randint(low, high + 1, shape, generator=gen, device="cuda").float())


def prepare(case: dict, seed: int) -> SimpleNamespace:
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"append": _prepare_append, "attend": _prepare_attend, "step": _prepare_step, "select": _prepare_select, "reorder": _prepare_reorder}[case["kind"]]
    return make(case, rng, gen)


def _prepare_append(case: dict, rng, gen) -> SimpleNamespace:
    kv_heads, dim, block, io = case["kv_heads"], case["dim"], case["block"], DTYPES[case["io"]]
    rows = np.concatenate([np.full(case["chunks"], case["chunk"]), np.ones(case["seqs"], np.int64)]).astype(np.int64)
    before = np.concatenate([rng.integers(0, 100, case["chunks"]), rng.integers(case["low"] - 1, case["high"], case["seqs"])]).astype(np.int64)
    used = -(-(before + rows) // block)
    blocks = case["chunks"] * -(-(100 + case["chunk"]) // block) + case["seqs"] * -(-case["high"] // block) + 8
    ids = rng.permutation(blocks)
    starts = np.concatenate([[0], np.cumsum(rows)])
    seq = np.repeat(np.arange(rows.size), rows)
    where = before[seq] + np.arange(starts[-1]) - starts[seq]
    slots = ids[(np.cumsum(used) - used)[seq] + where // block] * block + where % block
    tokens = int(starts[-1])
    # The parts of one fused projection's output: strided rows; some tokens are larger than others.
    fused = _normal(gen, (tokens, 2 * kv_heads * dim), torch.float32)
    fused = (fused * torch.exp2(torch.randn((tokens, 1), generator=gen, device="cuda"))).to(io)
    shape, scales = (blocks, block, kv_heads, dim), (blocks, kv_heads)
    return SimpleNamespace(kind="append", keys=fused[:, : kv_heads * dim].view(tokens, kv_heads, dim), values=fused[:, kv_heads * dim :].view(tokens, kv_heads, dim),
                           slots=_device(slots, torch.int64), key_pool=_codes(gen, shape), value_pool=_codes(gen, shape),
                           key_scales=_scales(gen, scales, -8, -6), value_scales=_scales(gen, scales, -8, -6))  # fmt: skip


def _prepare_attend(case: dict, rng, gen) -> SimpleNamespace:
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    offsets = rng.integers(0, case["offset"] + 1, case["chunks"])
    contexts = np.concatenate([offsets + case["chunk"], rng.integers(case["low"], case["high"] + 1, case["seqs"])]).astype(np.int64)
    rows = np.concatenate([np.full(case["chunks"], case["chunk"]), np.ones(case["seqs"], np.int64)]).astype(np.int64)
    starts = np.concatenate([[0], np.cumsum(rows)])
    query_seq = np.repeat(np.arange(rows.size), rows)
    positions = np.arange(starts[-1]) - starts[query_seq] + (contexts - rows)[query_seq]
    used = -(-contexts // block)
    blocks = int(used.sum()) + 8
    ids = rng.permutation(blocks)
    tables = np.zeros((rows.size, int(used.max())), np.int64)
    tables[np.arange(tables.shape[1])[None, :] < used[:, None]] = ids[: int(used.sum())]
    pool, scales = (blocks, block, kv_heads, dim), (blocks, kv_heads)
    return SimpleNamespace(kind="attend", queries=_normal(gen, (int(starts[-1]), heads, dim), DTYPES[case["io"]]), positions=_device(positions, torch.int32),
                           query_seq=_device(query_seq, torch.int32), keys=_codes(gen, pool), values=_codes(gen, pool), key_scales=_scales(gen, scales, -8, -6),
                           value_scales=_scales(gen, scales, -8, -6), tables=_device(tables, torch.int32), contexts=_device(contexts, torch.int32), scale=dim**-0.5,
                           window=case["window"] or None, sinks=case["sinks"], max_context=int(contexts.max()), max_rows=int(rows.max()))  # fmt: skip


def _prepare_step(case: dict, rng, gen) -> SimpleNamespace:
    block, width = case["block"], case["width"]
    query = np.concatenate([np.full(case["chunks"], case["chunk"]), np.ones(case["seqs"], np.int64)]).astype(np.int64)
    before = rng.integers(0, case["high"], query.size)
    before[rng.random(query.size) < 0.1] = 0  # new requests
    query[(rng.random(query.size) < 0.05) & (np.arange(query.size) > 0)] = 0  # requests that wait
    held = -(-before // block)
    taken = int(held.sum())
    need = int((-(-(before + query) // block) - held).sum())
    ids = rng.permutation(taken + need + 64)
    tables = np.zeros((query.size, width), np.int64)
    tables[np.arange(width)[None, :] < held[:, None]] = ids[:taken]
    # One step in eight finds fewer free blocks than it asks for.
    free = ids[taken : taken + (need * 7 // 8 if rng.random() < 0.125 else need + 32)]
    return SimpleNamespace(kind="step", query_lens=_device(query, torch.int32), contexts=_device(before + query, torch.int32), tables=_device(tables, torch.int32),
                           free=_device(free, torch.int32), next_free=torch.zeros(1, dtype=torch.int32, device="cuda"), block=block, rows=case["rows"])  # fmt: skip


def _prepare_select(case: dict, rng, gen) -> SimpleNamespace:
    rows, vocab, beams = case["groups"] * case["beams"], case["vocab"], case["beams"]
    # A decoder's logits: a broad bulk with some dozens of likely tokens above it, rows of different sharpness.
    logits = torch.randn((rows, vocab), generator=gen, device="cuda") * (1.0 + 1.5 * torch.rand((rows, 1), generator=gen, device="cuda"))
    stretch = vocab // 48  # a likely token in each: all at places of their own
    likely = torch.arange(48, device="cuda") * stretch + torch.randint(0, stretch, (rows, 48), generator=gen, device="cuda")
    logits.scatter_(1, likely, 6.0 + 6.0 * torch.rand((rows, 48), generator=gen, device="cuda"))
    scores = -torch.cumsum(torch.rand((case["groups"], beams), generator=gen, device="cuda"), dim=1) - 20 * torch.rand((case["groups"], 1), generator=gen, device="cuda")
    first = torch.rand((case["groups"], 1), generator=gen, device="cuda") < 0.1  # requests at their first token: one beam counts
    scores = torch.where(first & (torch.arange(beams, device="cuda") > 0), -math.inf, scores)
    finished = torch.rand(rows, generator=gen, device="cuda") < 0.1
    return SimpleNamespace(kind="select", logits=logits.to(DTYPES[case["io"]]), scores=scores.reshape(-1).contiguous(), finished=finished, beams=beams, count=case["count"],
                           end_token=int(rng.integers(0, vocab)))  # fmt: skip


def _prepare_reorder(case: dict, rng, gen) -> SimpleNamespace:
    groups, beams, layers, block, width = case["groups"], case["beams"], case["layers"], case["block"], case["width"]
    contexts = rng.integers(max(1, case["context"] * 3 // 4), case["context"] + 1, groups)
    used = -(-contexts // block)
    shared = np.maximum(contexts // block - rng.integers(0, 4, groups), 0)  # leading blocks that the group's beams share
    column = np.arange(width)
    own_blocks = int(((used - shared) * beams).sum())
    blocks = groups * (-(-case["context"] // block) + 4 * beams) + 4
    ids = rng.permutation(blocks)
    tables = np.zeros((groups, beams, width), np.int64)
    at = np.broadcast_to((column >= shared[:, None, None]) & (column < used[:, None, None]), tables.shape)
    tables[at] = ids[:own_blocks]
    for g in range(groups):
        tables[g, :, : shared[g]] = ids[own_blocks + int(shared[:g].sum()) :][: shared[g]]
    # Few beams carry on most continuations.
    parents = np.minimum(rng.geometric(0.4, (groups, beams)) - 1, beams - 1)
    shape, kv = (layers, blocks, block, case["kv_heads"], case["dim"]), {**DTYPES, "e4m3": E4M3}[case["cache"]]
    if case["cache"] == "e4m3":
        scales = (layers, blocks, case["kv_heads"])
        states = [_codes(gen, shape), _codes(gen, shape), _scales(gen, scales, -8, -6), _scales(gen, scales, -8, -6)]
    else:
        states = [torch.randn(shape, generator=gen, device="cuda", dtype=kv) for _ in range(2)]
    return SimpleNamespace(kind="reorder", tables=_device(tables.reshape(groups * beams, width), torch.int32), parents=_device(parents, torch.int32),
                           contexts=_device(contexts, torch.int32), states=states, block=block)  # fmt: skip


# --- one pass ---------------------------------------------------------------------------------


def run(s: SimpleNamespace):
    if s.kind == "append":
        return _own_append(s) if own else _plain_append(s)
    if s.kind == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    if s.kind == "step":
        return _own_step(s) if own else _plain_step(s)
    if s.kind == "select":
        return _own_select(s) if own else _plain_select(s)
    return _own_reorder(s) if own else _plain_reorder(s)


def _own_append(s):
    from paged_kv_serving_amd import ops

    ops.append_kv_e4m3(s.key_pool, s.value_pool, s.key_scales, s.value_scales, s.keys, s.values, s.slots)
    return s.key_pool, s.value_pool, s.key_scales, s.value_scales


def _own_attend(s):
    from paged_kv_serving_amd import ops

    return ops.paged_attention_e4m3(s.queries, s.positions, s.query_seq, s.keys, s.values, s.key_scales, s.value_scales, s.tables, s.contexts, s.scale,
                                    window=s.window, sinks=s.sinks, max_context_len=s.max_context, max_query_len=s.max_rows)  # fmt: skip


def _own_step(s):
    from paged_kv_serving_amd import ops

    step = ops.step_metadata(s.query_lens, s.contexts, s.tables, s.free, s.next_free, block_size=s.block, num_rows=s.rows)
    return step.query_seq, step.query_positions, step.positions, step.slot_mapping, step.query_starts, step.context_lens, step.next_free, s.tables


def _own_select(s):
    from paged_kv_serving_amd import ops

    best = ops.beam_select(s.logits, s.scores, num_beams=s.beams, count=s.count, finished=s.finished, end_token=s.end_token)
    return best.scores, best.beams, best.tokens


def _own_reorder(s):
    from paged_kv_serving_amd import ops

    return ops.beam_reorder(s.tables, s.parents, s.contexts, s.states, block_size=s.block), *s.states


def _plain_append(s):
    """Codes are returned in their own type, whose values they are, and each block's scale beside them."""
    block_size = s.key_pool.shape[1]
    block, offset = s.slots // block_size, s.slots % block_size
    # Tokens before the first one that is written stay; a block written from its start begins anew.
    first = torch.full((s.key_pool.shape[0],), block_size, device="cuda").scatter_reduce(0, block, offset, "amin")
    touched = torch.unique(block)
    stays = torch.arange(block_size, device="cuda") < first[touched, None]  # [touched, block_size]

    def put(pool, scales, new):
        new, held = new.float(), pool.view(torch.uint8)  # the codes' bytes
        most = torch.zeros(scales.shape, device="cuda").scatter_reduce(0, block[:, None].expand(-1, scales.shape[1]), new.abs().amax(-1), "amax")[touched]
        fraction, exponent = torch.frexp(most)  # most = fraction * 2^exponent; 448 is 0.875 * 2^9
        exponent = torch.where(fraction > LARGEST / 512, exponent - 8, exponent - 9).clamp(min=LOW_EXPONENT)
        need = torch.exp2(torch.where(most > 0, exponent, LOW_EXPONENT).float())
        before = scales[touched]
        after = torch.where(first[touched, None] > 0, torch.maximum(before, need), need)
        codes = held[touched]
        kept = (codes.view(E4M3).float() * (before / after)[:, None, :, None]).to(E4M3).view(torch.uint8)
        held[touched] = torch.where(stays[:, :, None, None], kept, codes)
        scales[touched] = after
        held.view(-1, *pool.shape[2:])[s.slots] = (new / scales[block][:, :, None]).to(E4M3).view(torch.uint8)

    put(s.key_pool, s.key_scales, s.keys)
    put(s.value_pool, s.value_scales, s.values)
    return s.key_pool, s.value_pool, s.key_scales, s.value_scales


def _plain_attend(s):
    """Every sequence's rows side by side (padded to the longest run), over the keys that any of them can see."""
    total, heads, dim = s.queries.shape
    seqs, (block, kv_heads) = s.tables.shape[0], s.keys.shape[1:3]
    where = torch.arange(total, device="cuda")
    seq = s.query_seq.long()
    first = torch.full((seqs,), total, device="cuda").scatter_reduce(0, seq, where, "amin")
    at = where - first[seq]  # the row's place among its sequence's
    q = torch.zeros((seqs, s.max_rows, heads, dim), device="cuda")
    q[seq, at] = s.queries.float()
    pos = torch.full((seqs, s.max_rows), -1, dtype=torch.int64, device="cuda")
    pos[seq, at] = s.positions.long()
    # Keys: the first `sinks` of the sequence, then its last window + max_rows.
    window = s.window or s.max_context
    span = min(window + s.max_rows - 1, s.max_context)
    begin = (s.contexts.long()[:, None] - span).clamp(min=0)
    key = torch.cat([torch.arange(s.sinks, device="cuda").expand(seqs, -1), begin + torch.arange(span, device="cuda")], dim=1)
    once = torch.cat([key[:, : s.sinks] < begin, key[:, s.sinks :] < s.contexts[:, None]], dim=1)
    key = key.clamp(max=s.max_context - 1)
    page = s.tables.long().gather(1, key // block)
    slot = page * block + key % block

    def values_of(pool, scales):  # [seqs, kv_heads, keys, dim]
        codes = pool.view(torch.uint8).view(-1, kv_heads, dim)[slot].view(E4M3)
        return (codes.float() * scales[page][..., None]).transpose(1, 2).contiguous()

    k, v = values_of(s.keys, s.key_scales), values_of(s.values, s.value_scales)
    q = q.view(seqs, s.max_rows, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    scores = torch.matmul(q * s.scale, k.transpose(2, 3).contiguous()).view(seqs, heads, s.max_rows, -1)
    seen = once[:, None, :] & (key[:, None, :] <= pos[:, :, None]) & ((key[:, None, :] > pos[:, :, None] - window) | (key[:, None, :] < s.sinks))
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    sums = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, kv_heads, -1, key.shape[1]), v).view(seqs, heads, s.max_rows, dim) / torch.where(sums > 0, sums, 1.0)
    return out.transpose(1, 2)[seq, at].to(s.queries.dtype)


def _plain_step(s):
    query, context, block, width = s.query_lens.long(), s.contexts.long(), s.block, s.tables.shape[1]
    start = context - query
    held, used = (start + block - 1) // block, (context + block - 1) // block
    ends = torch.cumsum(query, 0)
    fits = (used <= width) & (ends <= s.rows)
    need = torch.where(fits, used - held, 0)
    taken = torch.cumsum(need, 0)  # blocks, this request's among them
    available = s.free.shape[0] - s.next_free.long()
    served = fits & ((need == 0) | (taken <= available))
    # A table column that the request newly uses takes the next free block.
    column = torch.arange(width, device="cuda")
    new = served[:, None] & (column >= held[:, None]) & (column < used[:, None])
    fresh = torch.where(new, s.next_free + (taken - need - held)[:, None] + column, 0)
    s.tables.copy_(torch.where(new, torch.cat([s.free, s.free.new_zeros(1)])[fresh], s.tables))
    row = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(ends, row, right=True)
    inside = seq < query.shape[0]
    seq = seq.clamp(max=query.shape[0] - 1)
    live = inside & served[seq]
    position = torch.where(live, start[seq] + row - (ends - query)[seq], 0)
    slots = torch.where(live, s.tables[seq, position // block].long() * block + position % block, -1)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), ends]).clamp(max=s.rows)
    next_free = s.next_free + torch.where(served & (need > 0), taken, 0).amax()
    return (torch.where(live, seq, -1).int(), position.int(), position, slots, starts.int(), torch.where(served, context, start).int(), next_free.int(), s.tables)


def _plain_select(s):
    """Scores in 64 bits: a continuation is chosen by how it compares with others of nearly its score."""
    rows, vocab = s.logits.shape
    groups = rows // s.beams
    kept = min(s.count, vocab)
    ordered, ids = torch.sort(s.logits, dim=1, descending=True, stable=True)  # equal logits: the lowest id first
    wide = s.logits.double()
    most = wide.amax(1, keepdim=True)
    norm = most + torch.log(torch.exp(wide - most).sum(1, keepdim=True))
    scores = s.scores.double()[:, None] + (ordered[:, :kept].double() - norm)
    counts = torch.isfinite(s.scores) & torch.isfinite(norm[:, 0])
    # A finished beam goes on with the end token alone, at no cost.
    only = torch.where(torch.arange(kept, device="cuda") == 0, s.scores.double()[:, None], -math.inf)
    scores = torch.where(s.finished[:, None], torch.where(torch.isfinite(s.scores)[:, None], only, -math.inf), torch.where(counts[:, None], scores, -math.inf))
    tokens = torch.where(s.finished[:, None], s.end_token, ids[:, :kept])
    beam = (torch.arange(rows, device="cuda") % s.beams)[:, None].expand(-1, kept)
    best, at = torch.sort(scores.view(groups, -1), dim=1, descending=True, stable=True)  # equal scores: the lowest beam first
    best, at = best[:, : s.count], at[:, : s.count]
    nothing = best == -math.inf
    beams = torch.where(nothing, 0, beam.reshape(groups, -1).gather(1, at))
    return best.float(), beams.int(), torch.where(nothing, s.end_token, tokens.reshape(groups, -1).gather(1, at)).int()


def _plain_reorder(s):
    groups, beams = s.parents.shape
    tables = s.tables.view(groups, beams, -1)
    parents, row = s.parents.long(), torch.arange(beams, device="cuda")
    is_child = parents[:, :, None] == row  # [groups, child, parent]
    further = (torch.cumsum(is_child.int(), 1) * is_child).sum(2) > 1  # not its parent's first child
    childless = ~is_child.any(1)
    # The n-th further child takes over the last block of the n-th row without children.
    nth = torch.cumsum(further.int(), 1)
    donor = ((torch.cumsum(childless.int(), 1)[:, None, :] == nth[:, :, None]) & childless[:, None, :]).int().argmax(2)
    full, part = s.contexts.long() // s.block, s.contexts % s.block > 0
    column = torch.arange(tables.shape[2], device="cuda")
    from_parent = tables.gather(1, parents[:, :, None].expand(-1, -1, tables.shape[2]))
    last = full.clamp(max=tables.shape[2] - 1)[:, None, None].expand(-1, beams, 1)
    source = from_parent.gather(2, last)[:, :, 0]
    target = torch.where(further, tables.gather(1, donor[:, :, None].expand(-1, -1, tables.shape[2])).gather(2, last)[:, :, 0], source)
    here = part[:, None, None] & (column == full[:, None, None])
    new = torch.where(column < full[:, None, None], from_parent, torch.where(here, target[:, :, None], tables))
    source, target = (torch.where(part[:, None], t, 0).reshape(-1).long() for t in (source, target))

    def move(state):
        held = state.view(torch.uint8) if state.dtype == E4M3 else state
        held[:, target] = held[:, source]
        return state

    return new.reshape(s.tables.shape), *map(move, s.states)


# --- what a pass cannot do without --------------------------------------------------------------


def work(case: dict) -> dict:
    size = {"f32": 4, "bf16": 2, "e4m3": 1}
    if case["kind"] == "append":
        tokens = case["seqs"] + case["chunks"] * case["chunk"]
        blocks = case["seqs"] + case["chunks"] * -(-case["chunk"] // case["block"])
        each = 2 * case["kv_heads"] * case["dim"]
        return {"bytes": tokens * (each * (size[case["io"]] + 1) + 8) + blocks * 2 * case["kv_heads"] * 8, "flops": 2 * tokens * each}
    if case["kind"] == "step":
        requests = case["seqs"] + case["chunks"]
        return {"bytes": case["rows"] * (4 + 4 + 8 + 8) + requests * 20 + 4 * (case["chunks"] * case["chunk"] // case["block"] + requests), "flops": 8 * case["rows"]}
    if case["kind"] == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * size[case["io"]] + 5) + case["groups"] * case["count"] * 12, "flops": 3 * rows * case["vocab"]}
    if case["kind"] == "reorder":
        # Of the geometric parents above, this share of rows is a further child: its block is read and written.
        beams = case["beams"]
        chance = [0.4 * 0.6**k for k in range(beams - 1)] + [0.6 ** (beams - 1)]
        further = sum((1 - p) ** beams for p in chance)
        part = (case["block"] - 1) / case["block"]
        each = 2 * case["layers"] * (case["block"] * case["kv_heads"] * case["dim"] * size[case["cache"]] + (4 * case["kv_heads"] if case["cache"] == "e4m3" else 0))
        return {"bytes": int(case["groups"] * (2 * further * part * each + beams * (8 * case["width"] + 4))), "flops": 0}
    # Keys that some row of a sequence sees are read once; the mean context stands for the drawn ones.
    io, heads, kv_heads, dim = size[case["io"]], case["heads"], case["kv_heads"], case["dim"]
    chunk, most = case["chunk"], case["window"] + case["sinks"] if case["window"] else 1 << 30
    decode_keys = min((case["low"] + case["high"]) / 2, most)
    before = case["offset"] / 2
    seen = [min(before + i + 1, most) for i in range(chunk)]
    read = min(before + chunk, most + chunk - 1) if chunk else 0
    rows = case["seqs"] + case["chunks"] * chunk
    keys = case["seqs"] * decode_keys + case["chunks"] * read
    pairs = case["seqs"] * decode_keys + case["chunks"] * sum(seen)
    return {"bytes": int(2 * kv_heads * keys * (dim + 4 / case["block"]) + 2 * rows * heads * dim * io), "flops": int(4 * heads * dim * pairs)}


# --- the definitions, in 64 bits ------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    make = {"append": _exact_append, "attend": _exact_attend, "step": _exact_step, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]]
    return make(s)


def _nearest(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 number nearest to each double, ties to the even one: 3 bits behind the leading one, steps of 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    size = s.key_pool.shape[1]
    slots = s.slots.cpu().numpy()
    order = np.argsort(slots // size, kind="stable")
    blocks, starts = np.unique(slots[order] // size, return_index=True)
    ends = np.append(starts[1:], slots.size)
    # One block after the other, its tokens as a table padded with the block's first new token.
    count = ends - starts
    pick = order[starts[:, None] + np.minimum(np.arange(count.max()), count[:, None] - 1)]
    rows, block = torch.from_numpy(pick).cuda(), torch.from_numpy(blocks).cuda()
    first = torch.from_numpy(np.minimum.reduceat(slots[order] % size, starts)).cuda()
    out = []
    for pool, scales, new in ((s.key_pool, s.key_scales, s.keys), (s.value_pool, s.value_scales, s.values)):
        pool, scales, new = pool.float().double(), scales.double(), new.double()
        most = new.abs().amax(2)[rows].amax(1)
        need = torch.exp2(torch.ceil(torch.log2(most.clamp(min=1e-300) / LARGEST)).clamp(min=LOW_EXPONENT))
        need = torch.where(most <= LARGEST * need / 2, need / 2, torch.where(most > LARGEST * need, 2 * need, need))
        scale = torch.where(first[:, None] > 0, torch.maximum(scales[block], need), need)
        held = _nearest(pool[block] * scales[block][:, None, :, None] / scale[:, None, :, None])
        keep = torch.arange(size, device="cuda")[None, :] < first[:, None]
        pool[block] = torch.where(keep[:, :, None, None], held, pool[block])
        scales[block] = scale
        flat = pool.view(-1, *pool.shape[2:])
        flat[s.slots] = _nearest(new / scales[s.slots // size][:, :, None])
        out.append((pool, scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(s):
    out = torch.zeros(s.queries.shape, dtype=torch.float64, device="cuda")
    block, kv_heads, dim = s.keys.shape[1:]
    group = s.queries.shape[1] // kv_heads
    seq = s.query_seq.cpu().numpy()
    for index, context in enumerate(s.contexts.tolist()):
        rows = torch.from_numpy(np.flatnonzero(seq == index)).cuda()
        ids = s.tables[index, : -(-context // block)].long()
        k, v = (
            (pool.view(torch.uint8)[ids].view(E4M3).float().double() * scales[ids].double()[:, None, :, None]).view(-1, kv_heads, dim)[:context]
            for pool, scales in ((s.keys, s.key_scales), (s.values, s.value_scales))
        )
        key = torch.arange(context, device="cuda")
        back = s.positions[rows].long()[:, None] - key[None, :]  # how far behind the row a key lies
        hidden = back < 0
        if s.window is not None:
            hidden |= (back >= s.window) & (key[None, :] >= s.sinks)
        for h in range(s.queries.shape[1]):
            score = s.queries[rows, h].double() @ k[:, h // group].t() * s.scale
            out[rows, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ v[:, h // group]
    return out


def _exact_step(s):
    """Request by request on the host."""
    query, context, tables, free = s.query_lens.tolist(), s.contexts.tolist(), s.tables.cpu().numpy().copy(), s.free.tolist()
    seqs, positions, slots = np.full(s.rows, -1, np.int64), np.zeros(s.rows, np.int64), np.full(s.rows, -1, np.int64)
    starts, contexts = [0], []
    asked = taken = 0
    for i, (q, c) in enumerate(zip(query, context)):
        row, starts = starts[-1], starts + [starts[-1] + q]
        held, used = -(-(c - q) // s.block), -(-c // s.block)
        fits = used <= tables.shape[1] and row + q <= s.rows
        asked += used - held if fits else 0
        if not fits or (used > held and asked > len(free)):
            contexts.append(c - q)
            continue
        if used > held:
            tables[i, held:used] = free[asked - (used - held) : asked]
            taken = asked
        contexts.append(c)
        at = np.arange(c - q, c)
        seqs[row : row + q], positions[row : row + q] = i, at
        slots[row : row + q] = tables[i, at // s.block].astype(np.int64) * s.block + at % s.block
    as_int = lambda x: _device(np.asarray(x), torch.int32)  # noqa: E731
    return as_int(seqs), as_int(positions), _device(positions, torch.int64), _device(slots, torch.int64), as_int(np.minimum(starts, s.rows)), as_int(contexts), as_int([taken]), as_int(tables)


def _exact_select(s):
    """Row by row in NumPy."""
    logits, scores, finished = s.logits.float().cpu().numpy(), s.scores.double().cpu().numpy(), s.finished.cpu().numpy()
    out = ([], [], [])
    for first in range(0, len(logits), s.beams):
        found = []
        for b in range(s.beams):
            x, score = logits[first + b].astype(np.float64), scores[first + b]
            if not math.isfinite(score):
                continue
            if finished[first + b]:
                found.append((-score, b, 0.0, s.end_token))
                continue
            norm = np.logaddexp.reduce(np.sort(x))
            if math.isfinite(norm):
                top = np.argpartition(-x, min(s.count, x.size - 1))[: s.count] if s.count < x.size else np.arange(x.size)
                top = np.flatnonzero(x >= x[top].min())  # ties with the last one too
                found += [(-(score + (x[i] - norm)), b, -x[i], int(i)) for i in top if x[i] > -math.inf]
        found = (sorted(found) + [(math.inf, 0, 0.0, s.end_token)] * s.count)[: s.count]
        for column, values in zip(out, zip(*((-n, b, t) for n, b, _, t in found))):
            column.append(values)
    return _device(np.asarray(out[0]), torch.float64), _device(np.asarray(out[1]), torch.int32), _device(np.asarray(out[2]), torch.int32)


def _exact_reorder(s):
    """Group by group: what is returned are the inputs' own numbers, moved."""
    groups, beams = s.parents.shape
    old, parents, contexts = s.tables.cpu().numpy().reshape(groups, beams, -1), s.parents.tolist(), s.contexts.tolist()
    new, source, target = old.copy(), [], []
    for g in range(groups):
        full, part = divmod(contexts[g], s.block)
        idle = [r for r in range(beams) if r not in parents[g]]
        seen = set()
        for child, parent in enumerate(parents[g]):
            new[g, child, :full] = old[g, parent, :full]
            if part:
                keeper = parent if parent not in seen else idle.pop(0)
                new[g, child, full] = old[g, keeper, full]
                if keeper != parent:
                    source.append(old[g, parent, full])
                    target.append(old[g, keeper, full])
            seen.add(parent)
    for state in s.states:
        held = state.view(torch.uint8) if state.dtype == E4M3 else state
        if source:
            held[:, _device(np.asarray(target), torch.int64)] = held[:, _device(np.asarray(source), torch.int64)]
    return _device(new.reshape(s.tables.shape), torch.int32), *s.states
