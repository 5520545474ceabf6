"""rope_append_axes against float32 expressions (bit for bit) and against float64."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.window import axis_of_frequency

pytestmark = pytest.mark.gpu


def tables(rows, half):
    import torch

    angles = np.outer(np.arange(rows), 10_000.0 ** (-np.arange(half) / half))
    return torch.from_numpy(np.cos(angles).astype(np.float32)), torch.from_numpy(np.sin(angles).astype(np.float32))


def make(tokens, heads, kv_heads, dim, half, axes, io, kv, seed=0, rows=97, blocks=19, block=5):
    import torch

    gen = torch.Generator().manual_seed(seed)
    fused = torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=gen).to(io)
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    cos, sin = tables(rows, half)
    return {
        "queries": q.view(tokens, heads, dim), "keys": k.view(tokens, kv_heads, dim), "values": v.view(tokens, kv_heads, dim),
        "positions": torch.randint(0, rows, (axes, tokens), generator=gen), "cos": cos, "sin": sin,
        "key_pool": torch.randn((blocks, block, kv_heads, dim), generator=gen).to(kv),
        "value_pool": torch.randn((blocks, block, kv_heads, dim), generator=gen).to(kv),
        "slots": torch.randperm(blocks * block, generator=gen)[:tokens],
    }  # fmt: skip


def expect(d, sections, interleaved, dtype):
    """(rotated queries, key pool, value pool) with the expression evaluated in ``dtype``."""
    import torch

    half = d["cos"].shape[1]
    axis = torch.tensor(axis_of_frequency(sections, interleaved))
    where = d["positions"][axis].t()  # [T, half]
    safe = where.clamp(0, d["cos"].shape[0] - 1)
    cos, sin = (t.to(dtype).gather(0, safe)[:, None] for t in (d["cos"], d["sin"]))
    alive = ((d["positions"] >= 0) & (d["positions"] < d["cos"].shape[0])).all(0)

    def turn(x):
        x = x.to(dtype)
        lo, hi = x[..., :half], x[..., half : 2 * half]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 2 * half :]], -1)

    pools = []
    for pool, new in ((d["key_pool"], turn(d["keys"])), (d["value_pool"], d["values"].to(dtype))):
        out = pool.to(dtype) if dtype == torch.float64 else pool.clone()
        stored = alive & (d["slots"] >= 0) & (d["slots"] < pool.shape[0] * pool.shape[1])
        out.view(-1, *pool.shape[2:])[d["slots"][stored]] = new[stored].to(out.dtype)
        pools.append(out)
    q = turn(d["queries"])
    return (q if dtype == torch.float64 else q.to(d["queries"].dtype)), *pools, alive


def call(device, d, **more):
    from paged_kv_serving_amd import ops

    g = {k: v.to(device) for k, v in d.items()}
    # The three parts stay views of one fused projection.
    fused = d["queries"]._base.to(device)
    heads, kv_heads, dim = d["queries"].shape[1], d["keys"].shape[1], d["queries"].shape[2]
    q, k, v = fused.view(fused.shape[0], -1).split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    tokens = d["queries"].shape[0]
    positions = g["positions"] if "sections" in more else g["positions"][0].contiguous()
    out = ops.rope_append_axes(
        g["key_pool"], g["value_pool"], q.view(tokens, heads, dim), k.view(tokens, kv_heads, dim), v.view(tokens, kv_heads, dim), positions,
        g["cos"], g["sin"], g["slots"], **more,
    )  # fmt: skip
    return out.cpu(), g["key_pool"].cpu(), g["value_pool"].cpu()


def same(got, want):
    import torch

    assert got.dtype == want.dtype and torch.equal(got, want)


TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")]


@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half,sections,interleaved", [
    (1, 1, 1, 2, 1, None, False),
    (3, 4, 4, 32, 16, None, False),
    (7, 8, 2, 64, 32, None, False),
    (13, 14, 2, 64, 32, (10, 11, 11), False),
    (13, 14, 2, 64, 32, (12, 10, 10), True),
    (5, 8, 1, 128, 64, (16, 24, 24), False),
    (5, 32, 8, 128, 64, (24, 20, 20), True),
    (9, 6, 3, 128, 32, (16, 16), False),  # half of a head stays as it is
    (9, 6, 3, 80, 20, (5, 5, 5, 5), False),
    (11, 3, 1, 10, 3, (1, 2), False),  # no vector fits
    (4, 2, 2, 256, 128, (128,), False),
    (90, 4, 2, 16, 8, (0, 8), False),
])  # fmt: skip
def test_matches_the_float32_expression_bit_for_bit(device, io, kv, tokens, heads, kv_heads, dim, half, sections, interleaved):
    import torch

    io, kv = getattr(torch, io), getattr(torch, kv)
    axes = len(sections) if sections else 1
    d = make(tokens, heads, kv_heads, dim, half, axes, io, kv, seed=tokens + dim)
    more = {} if sections is None else {"sections": sections, "interleaved": interleaved}
    got = call(device, d, **more)
    want = expect(d, sections or (half,), interleaved, torch.float32)
    for a, b in zip(got, want):
        same(a, b)
    # Against float64: two products and a sum, 3 roundings of values of at most |lo c| + |hi s|, and the output's own.
    exact = expect(d, sections or (half,), interleaved, torch.float64)
    for a, b in zip(got, exact):
        size = 2 * d["queries"].abs().max().item() if a.shape == d["queries"].shape else 2 * d["keys"].abs().max().item()
        step = torch.finfo(a.dtype).eps / 2
        assert ((a.double() - b).abs() <= 3 * 2**-24 * size + step * b.abs() * 1.01).all()


def test_equals_rope_append(device):
    import torch

    from paged_kv_serving_amd import ops

    d = make(33, 8, 8, 64, 32, 1, torch.float32, torch.bfloat16)
    got = call(device, d)
    g = {k: v.to(device) for k, v in d.items()}
    rotated = ops.rope_append(g["key_pool"], g["value_pool"], g["queries"].contiguous(), g["keys"].contiguous(), g["values"].contiguous(),
                              g["positions"][0], g["cos"], g["sin"], g["slots"])  # fmt: skip
    for a, b in zip(got, (rotated, g["key_pool"], g["value_pool"])):
        same(a, b.cpu())


def test_in_place_and_strided_output(device):
    import torch

    from paged_kv_serving_amd import ops

    d = make(17, 4, 2, 64, 32, 1, torch.bfloat16, torch.bfloat16)
    want = expect(d, (32,), False, torch.float32)[0]
    g = {k: v.to(device) for k, v in d.items()}
    q = g["queries"].contiguous()
    out = ops.rope_append_axes(g["key_pool"], g["value_pool"], q, g["keys"], g["values"], g["positions"][0], g["cos"], g["sin"], g["slots"], out=q)
    assert out is q
    same(q.cpu(), want)
    wide = torch.zeros((17, 6, 64), dtype=torch.bfloat16, device=device)
    ops.rope_append_axes(g["key_pool"], g["value_pool"], d["queries"].to(device).contiguous(), g["keys"], g["values"], g["positions"][0], g["cos"], g["sin"],
                         g["slots"], out=wide[:, 1:5])  # fmt: skip
    same(wide[:, 1:5].cpu(), want)
    assert not wide[:, 0].any() and not wide[:, 5].any()


@pytest.mark.parametrize("shift", [1, 3])
def test_odd_addresses_take_the_element_path(device, shift):
    import torch

    from paged_kv_serving_amd import ops

    d = make(6, 4, 2, 32, 16, 1, torch.bfloat16, torch.bfloat16)
    want = expect(d, (16,), False, torch.float32)
    g = {k: v.to(device) for k, v in d.items()}
    q = torch.zeros(6 * 4 * 32 + shift, dtype=torch.bfloat16, device=device)[shift:].view(6, 4, 32)
    q.copy_(g["queries"])
    out = ops.rope_append_axes(g["key_pool"], g["value_pool"], q, g["keys"], g["values"], g["positions"][0], g["cos"], g["sin"], g["slots"])
    for a, b in zip((out, g["key_pool"], g["value_pool"]), want):
        same(a.cpu(), b)


def test_padding_slots_and_positions_outside_the_tables(device):
    """A slot outside the pool writes nothing there; a position outside the tables skips the token."""
    import torch

    d = make(8, 4, 2, 64, 32, 3, torch.float32, torch.float32, rows=50)
    d["slots"][2], d["slots"][5] = -1, 19 * 5
    d["positions"][1, 3], d["positions"][2, 6] = 50, -1
    want = expect(d, (10, 11, 11), False, torch.float32)
    g = {k: v.to(device) for k, v in d.items()}
    from paged_kv_serving_amd import ops

    out = torch.full((8, 4, 64), 7.0, device=device)
    ops.rope_append_axes(g["key_pool"], g["value_pool"], g["queries"], g["keys"], g["values"], g["positions"], g["cos"], g["sin"], g["slots"],
                         sections=(10, 11, 11), out=out)  # fmt: skip
    alive = want[3]
    assert alive.tolist() == [True, True, True, False, True, True, False, True]
    same(out.cpu()[alive], want[0][alive])
    assert (out.cpu()[~alive] == 7.0).all()
    same(g["key_pool"].cpu(), want[1])
    same(g["value_pool"].cpu(), want[2])


def test_positions_shared_by_all_axes(device):
    """One row of positions broadcast over the axes is one-axis rotation."""
    import torch

    d = make(21, 4, 1, 64, 32, 1, torch.bfloat16, torch.bfloat16)
    want = call(device, d)
    d["positions"] = d["positions"].expand(3, -1)
    from paged_kv_serving_amd import ops

    g = {k: v.to(device) for k, v in d.items() if k != "positions"}
    row = d["positions"][0].contiguous().to(device)
    out = ops.rope_append_axes(g["key_pool"], g["value_pool"], g["queries"], g["keys"], g["values"], row.expand(3, -1), g["cos"], g["sin"], g["slots"],
                               sections=(8, 12, 12))  # fmt: skip
    for a, b in zip((out, g["key_pool"], g["value_pool"]), want):
        same(a.cpu(), b)


def test_infinities_and_nan_stay_in_their_places(device):
    import torch

    d = make(4, 2, 1, 32, 16, 1, torch.bfloat16, torch.bfloat16)
    base = d["queries"]._base
    base[1, 3], base[2, 40], base[3, 70] = float("inf"), float("nan"), float("-inf")
    got, want = call(device, d), expect(d, (16,), False, torch.float32)
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0))


def test_captured_and_replayed(device):
    import torch

    from paged_kv_serving_amd import ops

    d = make(12, 8, 2, 64, 32, 3, torch.bfloat16, torch.bfloat16)
    g = {k: v.to(device).contiguous() for k, v in d.items()}
    out = torch.empty_like(g["queries"])
    run = lambda: ops.rope_append_axes(g["key_pool"], g["value_pool"], g["queries"], g["keys"], g["values"], g["positions"], g["cos"], g["sin"],
                                       g["slots"], sections=(12, 10, 10), out=out)  # noqa: E731 # fmt: skip
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(3):
        new = make(12, 8, 2, 64, 32, 3, torch.bfloat16, torch.bfloat16, seed=seed + 9)
        for name in d:
            g[name].copy_(new[name])
        graph.replay()
        torch.cuda.synchronize()
        want = expect(new, (12, 10, 10), False, torch.float32)
        for a, b in zip((out, g["key_pool"], g["value_pool"]), want):
            same(a.cpu(), b)


def test_no_tokens_and_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    d = make(4, 4, 2, 32, 16, 2, torch.float32, torch.float32)
    g = {k: v.to(device) for k, v in d.items()}

    def run(**change):
        more = {k: change.pop(k) for k in ("sections", "interleaved", "out") if k in change}
        a = {**g, **change}
        return ops.rope_append_axes(a["key_pool"], a["value_pool"], a["queries"], a["keys"], a["values"], a["positions"], a["cos"], a["sin"], a["slots"], **more)

    none = run(queries=g["queries"][:0], keys=g["keys"][:0], values=g["values"][:0], positions=g["positions"][0, :0], slots=g["slots"][:0])
    assert none.shape == (0, 4, 32)
    one = g["positions"][0].contiguous()
    for change in (
        {}, {"sections": (8, 9)}, {"sections": (16,)}, {"sections": (-1, 17)}, {"sections": (0, 16), "interleaved": True},
        {"positions": one, "sections": (8, 8)}, {"positions": one.int()}, {"positions": one[:3]}, {"positions": one, "slots": g["slots"].int()},
        {"positions": one, "keys": g["keys"].bfloat16()}, {"positions": one, "queries": g["queries"].half(), "keys": g["keys"].half(), "values": g["values"].half()},
        {"positions": one, "key_pool": g["key_pool"][:-1]}, {"positions": one, "cos": g["cos"].double()}, {"positions": one, "cos": g["cos"][:, :8]},
        {"positions": one, "values": g["values"][:, :1]}, {"positions": one, "out": g["queries"].bfloat16()}, {"positions": one, "queries": g["queries"].transpose(0, 1)},
        {"positions": one, "slots": g["slots"].cpu()}, {"positions": one, "key_pool": g["key_pool"].half(), "value_pool": g["value_pool"].half()},
    ):  # fmt: skip
        with pytest.raises(ValueError):
            run(**change)
