"""The operators of windowed, grouped-head serving and of sampling, as they are measured.

Three kinds of pass, each one call of a serving step:

    rope    ops.rope_append_axes: queries and keys rotated by positions of one or several axes
            (time, height, width), and keys and values appended to a paged cache of fewer heads
    window  ops.paged_attention_window: attention over that cache with a sliding window and a few
            first tokens that stay visible, decode rows and prompt chunks in one ragged batch
    sample  ops.sample_tokens: temperature, top-k, min-p and top-p, drawn with given numbers

Sizes are those of this repository's configurations, benchmark and tests (blocks of 16, chunks of
512, contexts up to 32,768, vocabularies of 50,257 and 128,256, heads of 64 and 128) and generic
ones between them.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ROPE_BASE = 10_000.0


def listed() -> list[dict]:
    return [
        # A decode step's append of a few interactive sequences. Latency.
        {"name": "rope_4_bf16", "kind": "rope", "tokens": 4, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1, "io": "bf16", "kv": "bf16", "block": 16,
         "pool": 4096},
        # The tokens of a full step of prompt chunks beside decode rows, everything float32.
        {"name": "rope_4216_f32", "kind": "rope", "tokens": 4216, "heads": 32, "kv_heads": 32, "dim": 128, "rotary": 128, "axes": 1, "io": "f32", "kv": "f32", "block": 16,
         "pool": 12288},
        # Image and video tokens of several prompts: three position axes, grouped heads.
        {"name": "rope_16384_axes_bf16", "kind": "rope", "tokens": 16384, "heads": 32, "kv_heads": 4, "dim": 128, "rotary": 128, "axes": 3, "io": "bf16", "kv": "bf16",
         "block": 16, "pool": 40960},
        # One interactive sequence with small heads and a short window. Latency.
        {"name": "window_decode_1", "kind": "window", "seqs": 1, "low": 1500, "high": 1500, "chunks": 0, "chunk": 0, "offset": 0, "heads": 8, "kv_heads": 2, "dim": 64,
         "window": 512, "sinks": 4, "io": "bf16", "kv": "bf16", "block": 16},
        # A decode step of 64 sequences, most of them longer than the window.
        {"name": "window_decode_64_bf16", "kind": "window", "seqs": 64, "low": 2048, "high": 16384, "chunks": 0, "chunk": 0, "offset": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 4096, "sinks": 4, "io": "bf16", "kv": "bf16", "block": 16},
        # The headline batch (64 sequences up to 4k, as many key heads as query heads, float32) under a window.
        {"name": "window_decode_64_f32", "kind": "window", "seqs": 64, "low": 512, "high": 4096, "chunks": 0, "chunk": 0, "offset": 0, "heads": 32, "kv_heads": 32,
         "dim": 128, "window": 1024, "sinks": 16, "io": "f32", "kv": "f32", "block": 16},
        # The prompt chunks of a full step, grouped heads.
        {"name": "window_prefill_8x512_bf16", "kind": "window", "seqs": 0, "low": 0, "high": 0, "chunks": 8, "chunk": 512, "offset": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "window": 1024, "sinks": 4, "io": "bf16", "kv": "bf16", "block": 16},
        # Odd-sized chunks beside decode rows, float32 activations over a bfloat16 cache.
        {"name": "window_mixed_2x301_24", "kind": "window", "seqs": 24, "low": 100, "high": 4000, "chunks": 2, "chunk": 301, "offset": 700, "heads": 16, "kv_heads": 16,
         "dim": 64, "window": 500, "sinks": 5, "io": "f32", "kv": "bf16", "block": 16},
        # One interactive sequence, a nucleus. Latency.
        {"name": "sample_1x32000", "kind": "sample", "rows": 1, "vocab": 32000, "io": "f32", "mode": "top_p", "per_row": False},
        # A decode step, top-k then a nucleus, an odd vocabulary.
        {"name": "sample_64x50257", "kind": "sample", "rows": 64, "vocab": 50257, "io": "f32", "mode": "top_k_p", "per_row": False},
        # A large decode step whose requests each bring their own settings.
        {"name": "sample_256x128256", "kind": "sample", "rows": 256, "vocab": 128256, "io": "f32", "mode": "mixed", "per_row": True},
        # bfloat16 logits (many ties) cut by min-p alone, rows of odd length.
        {"name": "sample_96x100003_bf16", "kind": "sample", "rows": 96, "vocab": 100003, "io": "bf16", "mode": "min_p", "per_row": False},
    ]  # fmt: skip


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    """One more case of the ranges above; none costs more than the largest listed ones."""
    kind = rng.choices(["rope", "window", "sample"], [3, 6, 5])[0]
    if kind == "sample":
        vocab = _log(rng, 200, 128256)
        return {"kind": kind, "rows": min(_log(rng, 1, 256), max(1, 256 * 128256 // vocab)), "vocab": vocab, "io": rng.choice(["f32", "f32", "bf16"]),
                "mode": rng.choice(["plain", "top_k", "top_p", "min_p", "top_k_p", "mixed"]), "per_row": rng.random() < 0.5}  # fmt: skip
    io, kv = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
    kv_heads, group = rng.choice([(1, 8), (2, 4), (2, 7), (4, 4), (4, 8), (8, 1), (8, 4), (16, 1), (8, 2), (1, 16)])
    dim = rng.choice([32, 64, 64, 128, 128, 128, 256]) if kv_heads * group <= 16 else rng.choice([32, 64, 128])
    shape = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "io": io, "kv": kv, "block": rng.choice([1, 7, 16, 16, 16, 32, 64])}
    if kind == "rope":
        rotary = dim if rng.random() < 0.7 else dim // 2
        tokens = _log(rng, 1, 8192)
        return {"kind": kind, "tokens": tokens, "rotary": rotary, "axes": rng.choice([1, 1, 3, 3, 2]), "pool": 2 * tokens + rng.randint(64, 4096), **shape}
    window, sinks = _log(rng, 16, 4096), rng.choice([0, 0, 1, 4, 4, 16, 64])
    row = 2 * kv_heads * dim * (4 if kv == "f32" else 2)
    high = _log(rng, 16, 16384)
    mode = rng.choice(["decode", "decode", "prefill", "mixed"])
    seqs = 0 if mode == "prefill" else min(_log(rng, 1, 64), max(1, 1_000_000_000 // (row * (min(high, window + sinks) + 1))), max(1, 4_000_000_000 // (row * high)))
    chunks = 0 if mode == "decode" else rng.randint(1, 8 if mode == "prefill" else 2)
    chunk = 0 if mode == "decode" else _log(rng, 2, 512)
    offset = 0 if mode == "decode" else _log(rng, 1, 4096) - 1
    while chunks * chunk * min(window + sinks, offset + chunk) > 4_000_000:  # (row, key) pairs of the largest listed case
        chunk = chunk * 3 // 4
    if mode == "mixed":  # the plain form pads every sequence to the longest run of rows
        seqs = min(seqs, max(1, 400_000_000 // (kv_heads * group * chunk * (window + sinks + chunk))))
    return {"kind": kind, "seqs": seqs, "low": max(1, int(high * rng.uniform(0.1, 1.0))) if seqs else 0, "high": high if seqs else 0, "chunks": chunks, "chunk": chunk,
            "offset": offset, "window": window, "sinks": sinks, **shape}  # fmt: skip


# --- inputs ----------------------------------------------------------------------------------


def _normal(gen: torch.Generator, shape, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _device(array, dtype) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(array)).to(dtype).cuda()


def prepare(case: dict, seed: int) -> SimpleNamespace:
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"rope": _prepare_rope, "window": _prepare_window, "sample": _prepare_sample}[case["kind"]]
    return make(case, rng, gen)


def _prepare_rope(case: dict, rng, gen) -> SimpleNamespace:
    tokens, heads, kv_heads, dim, half = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rotary"] // 2
    io, kv, block = DTYPES[case["io"]], DTYPES[case["kv"]], case["block"]
    # The three parts of one fused projection's output: strided rows, as a model has them.
    fused = _normal(gen, (tokens, (heads + 2 * kv_heads) * dim), io)
    queries = fused[:, : heads * dim].view(tokens, heads, dim)
    keys = fused[:, heads * dim : (heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    values = fused[:, (heads + kv_heads) * dim :].view(tokens, kv_heads, dim)
    rows = 8192
    angles = np.outer(np.arange(rows, dtype=np.float64), ROPE_BASE ** (-np.arange(half, dtype=np.float64) / half))
    slots = rng.permutation(-(-case["pool"] // block) * block)[:tokens]
    if case["axes"] == 1:
        positions = rng.integers(0, rows - 1) - np.arange(tokens)[::-1] % rows
        positions, sections = np.where(positions < 0, positions + rows, positions), None
    else:  # frames of a video: time, height and width of each token
        width = int(rng.integers(12, 40))
        where = np.arange(tokens)
        positions = np.stack([where // (width * width) % rows, where // width % width, where % width])[: case["axes"]]
        rest = half - half // 4
        sections = (half // 4, rest - rest // 2, rest // 2)[:3] if case["axes"] == 3 else (half - half // 2, half // 2)
    pool = (-(-case["pool"] // block), block, kv_heads, dim)
    return SimpleNamespace(kind="rope", queries=queries, keys=keys, values=values, positions=_device(positions, torch.int64), sections=sections,
                           cos=_device(np.cos(angles), torch.float32), sin=_device(np.sin(angles), torch.float32),
                           key_pool=_normal(gen, pool, kv), value_pool=_normal(gen, pool, kv), slots=_device(slots, torch.int64))  # fmt: skip


def _prepare_window(case: dict, rng, gen) -> SimpleNamespace:
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    io, kv = DTYPES[case["io"]], DTYPES[case["kv"]]
    chunk_offsets = rng.integers(0, case["offset"] + 1, case["chunks"])
    contexts = np.concatenate([chunk_offsets + case["chunk"], rng.integers(case["low"], case["high"] + 1, case["seqs"])]).astype(np.int64)
    rows = np.concatenate([np.full(case["chunks"], case["chunk"]), np.ones(case["seqs"], np.int64)]).astype(np.int64)
    starts = np.concatenate([[0], np.cumsum(rows)])
    query_seq = np.repeat(np.arange(rows.size), rows)
    positions = np.arange(starts[-1]) - starts[query_seq] + (contexts - rows)[query_seq]
    used = -(-contexts // block)
    blocks = int(used.sum()) + 8
    ids = rng.permutation(blocks)
    tables = np.zeros((rows.size, int(used.max())), np.int64)
    tables[np.arange(tables.shape[1])[None, :] < used[:, None]] = ids[: int(used.sum())]
    pool = (blocks, block, kv_heads, dim)
    return SimpleNamespace(kind="window", queries=_normal(gen, (int(starts[-1]), heads, dim), io), positions=_device(positions, torch.int32),
                           query_seq=_device(query_seq, torch.int32), keys=_normal(gen, pool, kv), values=_normal(gen, pool, kv),
                           tables=_device(tables, torch.int32), contexts=_device(contexts, torch.int32), scale=dim**-0.5, window=case["window"],
                           sinks=case["sinks"], max_context=int(contexts.max()), max_rows=int(rows.max()))  # fmt: skip


def _prepare_sample(case: dict, rng, gen) -> SimpleNamespace:
    rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
    # A decoder's logits: a broad bulk with some dozens of likely tokens above it, rows of different sharpness.
    logits = torch.randn((rows, vocab), generator=gen, device="cuda") * (1.0 + 1.5 * torch.rand((rows, 1), generator=gen, device="cuda"))
    likely = torch.randint(0, vocab, (rows, 48), generator=gen, device="cuda")
    logits.scatter_(1, likely, 6.0 + 6.0 * torch.rand((rows, 48), generator=gen, device="cuda"))

    def setting(name, values, dtype):
        """One value for the batch, or one for each row; `mixed` gives a row any of them."""
        if case["per_row"] or mode == "mixed":
            return _device(rng.choice(np.asarray(values), rows), dtype)
        return values[int(rng.integers(len(values)))]

    off = {"top_k": [0], "top_p": [1.0], "min_p": [0.0]}
    some = {"top_k": [1, 20, 50, 200, 1000], "top_p": [0.5, 0.8, 0.9, 0.95], "min_p": [0.02, 0.05, 0.1]}
    used = {"plain": (), "top_k": ("top_k",), "top_p": ("top_p",), "min_p": ("min_p",), "top_k_p": ("top_k", "top_p"), "mixed": ("top_k", "top_p", "min_p")}[mode]
    temperature = setting("temperature", [0.0, 0.6, 0.8, 1.0, 1.3] if mode == "mixed" else [0.6, 0.8, 1.0, 1.3], torch.float32)
    values = {name: (some[name] + off[name] if mode == "mixed" else some[name]) if name in used else off[name] for name in off}
    return SimpleNamespace(kind="sample", logits=logits.to(DTYPES[case["io"]]), uniforms=torch.rand(rows, generator=gen, device="cuda"), temperature=temperature,
                           top_k=setting("top_k", values["top_k"], torch.int32), top_p=setting("top_p", values["top_p"], torch.float32),
                           min_p=setting("min_p", values["min_p"], torch.float32))  # fmt: skip


# --- one pass ---------------------------------------------------------------------------------


def run(s: SimpleNamespace):
    if s.kind == "rope":
        return _own_rope(s) if own else _plain_rope(s)
    if s.kind == "window":
        return _own_window(s) if own else _plain_window(s)
    return _own_sample(s) if own else _plain_sample(s)


def _own_rope(s):
    from paged_kv_serving_amd import ops

    rotated = ops.rope_append_axes(s.key_pool, s.value_pool, s.queries, s.keys, s.values, s.positions, s.cos, s.sin, s.slots, sections=s.sections)
    return rotated, s.key_pool, s.value_pool


def _own_window(s):
    from paged_kv_serving_amd import ops

    return ops.paged_attention_window(s.queries, s.positions, s.query_seq, s.keys, s.values, s.tables, s.contexts, s.scale, window=s.window, sinks=s.sinks,
                                      max_context_len=s.max_context, max_query_len=s.max_rows)  # fmt: skip


def _own_sample(s):
    from paged_kv_serving_amd import ops

    return ops.sample_tokens(s.logits, s.uniforms, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)


def _plain_rope(s):
    half = s.cos.shape[1]
    if s.sections is None:
        cos, sin = s.cos[s.positions], s.sin[s.positions]
    else:  # frequency i turns by the position of the axis whose section it lies in
        axis = torch.repeat_interleave(torch.arange(len(s.sections), device="cuda"), torch.tensor(s.sections, device="cuda"), output_size=half)
        where = s.positions[axis].t()
        cos, sin = s.cos.gather(0, where), s.sin.gather(0, where)
    cos, sin = cos[:, None, :], sin[:, None, :]

    def turn(x):
        x = x.float()
        low, high, rest = x[..., :half], x[..., half : 2 * half], x[..., 2 * half :]
        return torch.cat([low * cos - high * sin, high * cos + low * sin, rest], dim=-1)

    pool = (-1, *s.key_pool.shape[2:])
    s.key_pool.view(pool)[s.slots] = turn(s.keys).to(s.key_pool.dtype)
    s.value_pool.view(pool)[s.slots] = s.values.to(s.value_pool.dtype)
    return turn(s.queries).to(s.queries.dtype), s.key_pool, s.value_pool


def _plain_window(s):
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
    span = min(s.window + s.max_rows - 1, s.max_context)
    begin = (s.contexts.long()[:, None] - span).clamp(min=0)
    key = torch.cat([torch.arange(s.sinks, device="cuda").expand(seqs, -1), begin + torch.arange(span, device="cuda")], dim=1)
    once = torch.cat([key[:, : s.sinks] < begin, key[:, s.sinks :] < s.contexts[:, None]], dim=1)
    key = key.clamp(max=s.max_context - 1)
    slot = s.tables.long().gather(1, key // block) * block + key % block
    k = s.keys.view(-1, kv_heads, dim)[slot].float().transpose(1, 2).contiguous()  # [seqs, kv_heads, keys, dim]
    v = s.values.view(-1, kv_heads, dim)[slot].float().transpose(1, 2).contiguous()
    q = q.view(seqs, s.max_rows, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    scores = torch.matmul(q * s.scale, k.transpose(2, 3).contiguous()).view(seqs, heads, s.max_rows, -1)
    seen = once[:, None, :] & (key[:, None, :] <= pos[:, :, None]) & ((key[:, None, :] > pos[:, :, None] - s.window) | (key[:, None, :] < s.sinks))
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    sums = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, kv_heads, -1, key.shape[1]), v).view(seqs, heads, s.max_rows, dim) / torch.where(sums > 0, sums, 1.0)
    return out.transpose(1, 2)[seq, at].to(s.queries.dtype)


def _plain_sample(s):
    """Sums in 64 bits: a token is chosen by where a cumulative sum passes a number."""
    rows, vocab = s.logits.shape

    def column(value):
        value = value if isinstance(value, torch.Tensor) else torch.full((rows,), value, device="cuda")
        return value.double()[:, None]

    temperature, top_k, top_p, min_p = column(s.temperature), column(s.top_k), column(s.top_p), column(s.min_p)
    if not isinstance(s.top_p, torch.Tensor):
        top_p, min_p = top_p.float().double(), min_p.float().double()
    ordered, ids = torch.sort(s.logits, dim=1, descending=True, stable=True)  # equal logits: the lowest id first
    ordered = ordered.double()
    weights = torch.exp((ordered - ordered[:, :1]) / torch.where(temperature > 0, temperature.float().double(), 1.0))
    rank = torch.arange(vocab, device="cuda")
    kept = ((top_k <= 0) | (rank < top_k)) & (weights >= min_p)
    mass = torch.cumsum(torch.where(kept, weights, 0.0), dim=1)
    last = torch.minimum((mass < top_p * mass[:, -1:]).sum(1, keepdim=True), kept.sum(1, keepdim=True) - 1)
    drawn = (mass <= s.uniforms.double()[:, None] * mass.gather(1, last)).sum(1, keepdim=True)
    drawn = torch.where(temperature > 0, torch.minimum(drawn, last), 0)
    return ids.gather(1, drawn)[:, 0].int()


# --- what a pass cannot do without --------------------------------------------------------------


def work(case: dict) -> dict:
    size = {"f32": 4, "bf16": 2}
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size[case["io"]] + 8), "flops": 2 * case["rows"] * case["vocab"]}
    io, kv, heads, kv_heads, dim = size[case["io"]], size[case["kv"]], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        each = 2 * heads * dim * io + 2 * kv_heads * dim * (io + kv) + 8 * (case["axes"] + 1) + 4 * case["rotary"]
        return {"bytes": case["tokens"] * each, "flops": case["tokens"] * 3 * (heads + kv_heads) * case["rotary"]}
    # Keys that some row of a sequence sees are read once; the mean context stands for the drawn ones.
    window, sinks, chunk = case["window"], case["sinks"], case["chunk"]
    decode_keys = min((case["low"] + case["high"]) / 2, window + sinks)
    before = case["offset"] / 2
    seen = [min(before + i + 1, window + sinks) for i in range(chunk)]
    read = min(before + chunk, window + sinks + chunk - 1) if chunk else 0
    rows = case["seqs"] + case["chunks"] * chunk
    pairs = case["seqs"] * decode_keys + case["chunks"] * sum(seen)
    return {"bytes": int(2 * kv_heads * dim * kv * (case["seqs"] * decode_keys + case["chunks"] * read) + 2 * rows * heads * dim * io), "flops": int(4 * heads * dim * pairs)}


# --- the definitions, in 64 bits ------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s)
    if case["kind"] == "window":
        return _exact_window(s)
    return _exact_sample(s)


def _exact_rope(s):
    half = s.cos.shape[1]
    positions = s.positions if s.sections is not None else s.positions[None]
    ends = np.cumsum(s.sections) if s.sections is not None else np.asarray([half])
    angle = [positions[int(np.searchsorted(ends, i, side="right"))] for i in range(half)]
    turn = torch.stack([torch.complex(s.cos[p, i].double(), s.sin[p, i].double()) for i, p in enumerate(angle)], dim=1)[:, None]

    def rotate(x):
        x = x.double()
        pair = torch.complex(x[..., :half].contiguous(), x[..., half : 2 * half].contiguous()) * turn
        x = x.clone()
        x[..., :half], x[..., half : 2 * half] = pair.real, pair.imag
        return x

    pools = []
    for pool, new in ((s.key_pool, rotate(s.keys)), (s.value_pool, s.values.double())):
        pool = pool.double()
        pool.view(-1, *pool.shape[2:])[s.slots] = new
        pools.append(pool)
    return rotate(s.queries), pools[0], pools[1]


def _exact_window(s):
    out = torch.zeros(s.queries.shape, dtype=torch.float64, device="cuda")
    block, kv_heads, dim = s.keys.shape[1:]
    group = s.queries.shape[1] // kv_heads
    seq = s.query_seq.cpu().numpy()
    for index, context in enumerate(s.contexts.tolist()):
        rows = torch.from_numpy(np.flatnonzero(seq == index)).cuda()
        ids = s.tables[index, : -(-context // block)].long()
        k = s.keys[ids].view(-1, kv_heads, dim)[:context].double()
        v = s.values[ids].view(-1, kv_heads, dim)[:context].double()
        key = torch.arange(context, device="cuda")
        back = s.positions[rows].long()[:, None] - key[None, :]  # how far behind the row a key lies
        hidden = (back < 0) | ((back >= s.window) & (key[None, :] >= s.sinks))
        for h in range(s.queries.shape[1]):
            score = s.queries[rows, h].double() @ k[:, h // group].t() * s.scale
            out[rows, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ v[:, h // group]
    return out


def _exact_sample(s):
    """Row by row in NumPy. The order of the tokens is that of their logits, ties by id."""
    logits = s.logits.float().cpu().numpy()
    rows, vocab = logits.shape

    def each(value, dtype):
        return value.cpu().numpy() if isinstance(value, torch.Tensor) else np.full(rows, value, dtype)

    temperature, top_k = each(s.temperature, np.float32), each(s.top_k, np.int32)
    top_p, min_p, uniforms = each(s.top_p, np.float32), each(s.min_p, np.float32), s.uniforms.cpu().numpy()
    out = np.zeros(rows, np.int32)
    for r in range(rows):
        order = np.lexsort((np.arange(vocab), -logits[r]))
        if temperature[r] <= 0:
            out[r] = order[0]
            continue
        x = logits[r][order].astype(np.float64)
        w = np.exp((x - x[0]) / np.float64(temperature[r]))
        count = min(int(top_k[r]) or vocab, int(np.count_nonzero(w >= np.float64(min_p[r]))))
        mass = np.cumsum(w[:count])
        last = min(int(np.searchsorted(mass, np.float64(top_p[r]) * mass[-1], side="left")), count - 1)
        out[r] = order[min(int(np.searchsorted(mass, np.float64(uniforms[r]) * mass[last], side="right")), last)]
    return torch.from_numpy(out).cuda()
