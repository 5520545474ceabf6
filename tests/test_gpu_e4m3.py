"""append_kv_e4m3 and paged_attention_e4m3 against the float64 definitions, at the sizes and masks where they can go
wrong."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import e4m3
from oracle.window import window_attention

pytestmark = pytest.mark.gpu

CAUSAL = 1 << 30


def codes_of(x):
    """float8_e4m3fn of numbers that the format holds (NaN among them)."""
    import torch

    return torch.from_numpy(np.asarray(x, np.float32)).to(torch.float8_e4m3fn)


def numbers(codes) -> np.ndarray:
    return codes.float().cpu().numpy().astype(np.float64)


# --- the append -------------------------------------------------------------------------------


def pool_of(blocks, block, heads, dim, seed):
    """Codes and scales as appends leave them."""
    rng = np.random.default_rng(seed)
    return e4m3.nearest(np.clip(rng.standard_normal((blocks, block, heads, dim)) * 110, -e4m3.LARGEST, e4m3.LARGEST)), np.exp2(rng.integers(-9, -5, (blocks, heads)).astype(np.float64))


def append(device, pools, keys, values, slots):
    """The call on device copies of ``pools`` = (key codes, key scales, value codes, value scales); what they hold then."""
    import torch

    from paged_kv_serving_amd import ops

    k, ks, v, vs = pools
    held = [codes_of(k).to(device), codes_of(v).to(device), *(torch.from_numpy(s.astype(np.float32)).to(device) for s in (ks, vs))]
    ops.append_kv_e4m3(*held, keys, values, torch.as_tensor(np.asarray(slots), dtype=torch.int64).to(device))
    return numbers(held[0]), held[2].double().cpu().numpy(), numbers(held[1]), held[3].double().cpu().numpy()


def check_append(device, pools, keys, values, slots):
    got = append(device, pools, keys.to(device), values.to(device), slots)
    want = [x.copy() for x in pools]
    e4m3.append(want[0], want[1], keys.float().numpy(), slots)
    e4m3.append(want[2], want[3], values.float().numpy(), slots)
    # What lies behind a written place counts as gone, and is left as it was here as there.
    for a, b, name in zip(got, want, ("keys", "key scales", "values", "value scales")):
        np.testing.assert_array_equal(a, b, err_msg=name)


def tokens_of(count, heads, dim, io, seed, spread=1.5):
    import torch

    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((count, heads, dim), generator=gen) * torch.exp2(spread * torch.randn((count, 1, 1), generator=gen))
    return x.to(getattr(torch, io))


def run_slots(runs, block, seed):
    """Slots of ``runs`` = (tokens, tokens before them), each in blocks of its own in a random order, and the blocks."""
    used = [-(-(n + before) // block) for n, before in runs]
    ids = np.random.default_rng(seed).permutation(sum(used) + 2)
    slots, at = [], 0
    for (n, before), count in zip(runs, used):
        where = np.arange(before, before + n)
        slots.append(ids[at + where // block] * block + where % block)
        at += count
    return np.concatenate(slots), sum(used) + 2


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("block", [1, 3, 16, 33, 128])
def test_appends_of_many_lengths(device, io, dim, block):
    runs = [(1, 0), (1, 1), (1, block - 1), (2, 2 * block - 1), (block, 0), (block, block // 2), (3 * block + 1, 5), (40, 7), (1, 3 * block)]
    slots, blocks = run_slots(runs, block, dim + block)
    heads = 3
    keys, values = (tokens_of(slots.size, heads, dim, io, dim + block + i) for i in (0, 1))
    check_append(device, (*pool_of(blocks, block, heads, dim, 1), *pool_of(blocks, block, heads, dim, 2)), keys, values, slots)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("block", [17, 32, 64, 65, 200])
def test_long_runs_of_larger_blocks(device, io, dim, block):
    """Runs that a wavefront holds, just does not, and reads twice; from rows that are not 16-byte aligned too."""
    runs = [(n, before) for n in (16, 17, 31, 32, 33, 63, 64, 65, 2 * block + 3) for before in (0, block - 5)] + [(1, 3)] * 4
    slots, blocks = run_slots(runs, block, dim + block)
    pools = (*pool_of(blocks, block, 2, dim, 1), *pool_of(blocks, block, 2, dim, 2))
    keys, values = (tokens_of(slots.size, 2, dim, io, dim + block + i) for i in (0, 1))
    check_append(device, pools, keys, values, slots)
    wide = keys.new_zeros((2, slots.size, 2 * dim + 1), device=device)
    for i, x in enumerate((keys, values)):
        wide[i, :, 1:] = x.flatten(1)
    apart = append(device, pools, *(x[:, 1:].unflatten(1, (2, dim)) for x in wide), slots)
    for a, b in zip(apart, append(device, pools, keys.to(device), values.to(device), slots)):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
def test_many_tokens_and_heads(device, io):
    """More tokens than one wavefront looks at, runs that lie across its window's ends."""
    runs = [(1, b) for b in range(60)] + [(301, 9), (512, 0), (300, 31)] + [(1, b) for b in range(30)]
    slots, blocks = run_slots(runs, 16, 3)
    slots[[7, 200, 700]] = -1, blocks * 16, 1 << 40  # padding; the second and third cut a run in two
    # A cut run's two parts share a block: parts are written by calls of their own.
    cut = [0, 200, 201, 700, 701, slots.size]
    heads, dim = 16, 128
    keys, values = (tokens_of(slots.size, heads, dim, io, i) for i in (0, 1))
    pools = (*pool_of(blocks, 16, heads, dim, 1), *pool_of(blocks, 16, heads, dim, 2))
    for a, b in zip(cut[:-1], cut[1:]):
        got = append(device, pools, keys[a:b].to(device), values[a:b].to(device), slots[a:b])
        for pool, scale, new in ((0, 1, keys), (2, 3, values)):
            e4m3.append(pools[pool], pools[scale], new[a:b].float().numpy(), slots[a:b])
        for x, y in zip(got, pools):
            np.testing.assert_array_equal(x, y)


def test_a_block_filled_by_many_calls(device):
    """Scales that grow from call to call, codes that are scaled down several times, a block that begins anew."""
    import torch

    heads, dim, block = 2, 64, 16
    keys, values = tokens_of(40, heads, dim, "float32", 5, spread=4.0), tokens_of(40, heads, dim, "float32", 6, spread=4.0)
    pools = (*pool_of(4, block, heads, dim, 3), *pool_of(4, block, heads, dim, 4))
    at = 0
    for count in (1, 1, 3, 1, 7, 12, 1, 14):
        slots = 16 + (np.arange(at, at + count) % 40)
        want = [x.copy() for x in pools]
        e4m3.append(want[0], want[1], keys[at : at + count].numpy(), slots)
        e4m3.append(want[2], want[3], values[at : at + count].numpy(), slots)
        got = append(device, pools, keys[at : at + count].to(device), values[at : at + count].to(device), slots)
        for x, y in zip(got, want):
            np.testing.assert_array_equal(x, y)
        pools, at = got, at + count
    assert torch.isfinite(torch.from_numpy(pools[0])).all()


def test_extreme_values(device):
    """Zeros, the smallest and largest numbers, values at a scale's border, what is not finite."""
    import torch

    rows = torch.zeros((12, 1, 32))
    rows[1] = 1e-45
    rows[2] = 448.0 * 2.0**-100
    rows[3] = torch.tensor(448.0 * 2.0**-100).nextafter(torch.tensor(1.0))
    rows[4], rows[5] = 3.5, torch.tensor(3.5).nextafter(torch.tensor(4.0))
    rows[6] = -(2.0**126)
    rows[7, 0, 3], rows[7, 0, 4:] = float("inf"), 2.0
    rows[8, 0, 5], rows[8, 0, 6:] = float("nan"), -3.0
    rows[9] = float("-inf")
    rows[10] = torch.linspace(-1.0, 1.0, 32)
    rows[11] = 464.0 / 448.0  # rounds to the largest code or the next scale's
    slots = np.arange(12)
    check_append(device, (*pool_of(12, 1, 1, 32, 0), *pool_of(12, 1, 1, 32, 1)), rows, rows.flip(0), slots)
    check_append(device, (*pool_of(3, 4, 1, 32, 0), *pool_of(3, 4, 1, 32, 1)), rows, rows.flip(0), slots)


def test_strided_unaligned_rows_and_an_empty_call(device):
    import torch

    heads, dim, block = 2, 64, 16
    slots, blocks = run_slots([(5, 3), (1, 0), (20, 10)], block, 2)
    for io in (torch.float32, torch.bfloat16):
        fused = torch.randn((slots.size, 3 * heads * dim + 1)).to(io)
        pools = (*pool_of(blocks, block, heads, dim, 1), *pool_of(blocks, block, heads, dim, 2))
        for start in (0, 1):  # 16-byte aligned rows (of some tokens), and rows aligned to an element only
            k, v = (fused[:, start + i * heads * dim :][:, : heads * dim].unflatten(1, (heads, dim)) for i in (0, 1))
            assert not k.is_contiguous()
            dense = append(device, pools, k.contiguous().to(device), v.contiguous().to(device), slots)
            f = fused.to(device)
            k, v = (f[:, start + i * heads * dim :][:, : heads * dim].unflatten(1, (heads, dim)) for i in (0, 1))
            for a, b in zip(append(device, pools, k, v, slots), dense):
                np.testing.assert_array_equal(a, b)
        none = torch.zeros((0, heads, dim), dtype=io, device=device)
        for a, b in zip(append(device, pools, none, none, []), pools):
            np.testing.assert_array_equal(a, b)


def test_append_past_32_bit_offsets(device):
    """A pool of more than 2^32 codes."""
    import torch

    from paged_kv_serving_amd import ops

    heads, dim, block = 8, 128, 16
    blocks = (1 << 32) // (heads * dim * block) + 20
    pool = [torch.zeros((blocks, block, heads, dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros((blocks, heads), device=device) for _ in range(2)]
    keys, values = tokens_of(20, heads, dim, "bfloat16", 1), tokens_of(20, heads, dim, "bfloat16", 2)
    slots = torch.arange((blocks - 2) * block, (blocks - 2) * block + 20)
    ops.append_kv_e4m3(*pool, *scales, keys.to(device), values.to(device), slots.to(device))
    for p, s, new in zip(pool, scales, (keys, values)):
        codes, scale = np.zeros((2, block, heads, dim)), np.zeros((2, heads))
        e4m3.append(codes, scale, new.float().numpy(), np.arange(20))
        tail = p.view(torch.uint8)[-2:].view(torch.float8_e4m3fn)
        np.testing.assert_array_equal(numbers(tail), codes)
        np.testing.assert_array_equal(s[-2:].double().cpu().numpy(), scale)
        assert not s[:-2].any()


def test_append_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    good = dict(
        key_pool=torch.zeros((3, 4, 2, 32), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
        value_pool=torch.zeros((3, 4, 2, 32), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
        key_scales=torch.zeros((3, 2), device=device), value_scales=torch.zeros((3, 2), device=device),
        keys=torch.ones((5, 2, 32), device=device), values=torch.ones((5, 2, 32), device=device),
        slot_mapping=torch.arange(5, device=device),
    )  # fmt: skip
    ops.append_kv_e4m3(**good)
    bad = [
        {"key_pool": good["key_pool"].float()}, {"value_pool": good["value_pool"].view(torch.uint8)}, {"key_pool": good["key_pool"][:2]},
        {"key_pool": good["key_pool"].transpose(0, 1)}, {"key_scales": good["key_scales"].double()}, {"value_scales": good["value_scales"][:2]},
        {"key_scales": torch.zeros((2, 3), device=device).t()}, {"keys": good["keys"].half()}, {"keys": good["keys"].bfloat16()}, {"keys": good["keys"][:4]},
        {"keys": good["keys"][:, :1], "values": good["values"][:, :1]}, {"keys": good["keys"][..., :16], "values": good["values"][..., :16]},
        {"keys": good["keys"].transpose(0, 1), "values": good["values"].transpose(0, 1)}, {"slot_mapping": good["slot_mapping"].int()},
        {"slot_mapping": good["slot_mapping"][:4]}, {"slot_mapping": good["slot_mapping"].cpu()}, {"values": good["values"].cpu()},
        {"slot_mapping": torch.arange(10, device=device)[::2]},
    ]  # fmt: skip
    for change in bad:
        with pytest.raises(ValueError):
            ops.append_kv_e4m3(**{**good, **change})
    with pytest.raises(ValueError, match="head_dim"):
        odd = torch.zeros((3, 4, 2, 48), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        ops.append_kv_e4m3(**{**good, "key_pool": odd, "value_pool": odd, "keys": torch.ones((5, 2, 48), device=device), "values": torch.ones((5, 2, 48), device=device)})


# --- the attention ------------------------------------------------------------------------------


def make(runs, heads, kv_heads, dim, block, io, seed=0):
    """A batch of ``runs`` = (rows, context) per sequence, each run's rows at its last positions."""
    import torch

    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    contexts = np.asarray([c for _, c in runs], np.int32)
    used = -(-contexts // block)
    blocks = int(used.sum()) + 3
    ids = rng.permutation(blocks)
    tables = np.full((len(runs), max(1, int(used.max())) + 2), -7, np.int32)  # past the used entries: anything
    at = 0
    for s, n in enumerate(used):
        tables[s, :n] = ids[at : at + n]
        at += n
    k, ks = pool_of(blocks, block, kv_heads, dim, seed + 1)
    v, vs = pool_of(blocks, block, kv_heads, dim, seed + 2)
    seqs = np.repeat(np.arange(len(runs)), [r for r, _ in runs]).astype(np.int32)
    return {
        "q": torch.randn((seqs.size, heads, dim), generator=gen).to(getattr(torch, io)), "k": k, "ks": ks, "v": v, "vs": vs,
        "positions": np.concatenate([np.arange(c - r, c) for r, c in runs]).astype(np.int32), "seqs": seqs, "tables": tables,
        "contexts": contexts, "scale": dim**-0.5,
    }  # fmt: skip


def call(device, d, window=None, sinks=0, **more):
    import torch

    from paged_kv_serving_amd import ops

    def put(x):
        return (x if isinstance(x, torch.Tensor) else torch.from_numpy(x)).to(device)

    more.setdefault("max_context_len", int(max(1, d["contexts"].max())))
    return ops.paged_attention_e4m3(put(d["q"]), put(d["positions"]), put(d["seqs"]), put(codes_of(d["k"])), put(codes_of(d["v"])),
                                    put(d["ks"].astype(np.float32)), put(d["vs"].astype(np.float32)), put(d["tables"]), put(d["contexts"]), d["scale"],
                                    window=window, sinks=sinks, **more)  # fmt: skip


def bound(d, want, size):
    """Of |out - want|. A score is a sum of dim products in float32: off by at most (dim + 4) 2^-24 of scale * sum |q k|,
    and bfloat16 pieces leave out 2^-24 of a product (codes times their scales are bfloat16 numbers). That moves a weight by
    twice as much, relatively; weights are rounded to 2^-17 at most where the output is bfloat16, sums of n terms to n
    2^-24; the output is a mean of values, rounded once to its type."""
    import torch

    keys = int(d["contexts"].max())
    values = e4m3.values(d["v"], d["vs"])
    most = np.abs(values[np.isfinite(values)]).max()
    scores = (d["q"].shape[2] + 8) * 2.0**-24 * size[..., None]
    off = most * (2 * np.expm1(2 * scores) + (keys + 16) * 2.0**-24)
    if d["q"].dtype == torch.bfloat16:
        off = off + most * 2.0**-16 + np.abs(want) * 2.0**-8
    return off


def check(device, d, window=None, sinks=0, **more):
    got = call(device, d, window, sinks, **more).float().cpu().numpy().astype(np.float64)
    want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                                  d["tables"], d["contexts"], d["scale"], window or CAUSAL, sinks)  # fmt: skip
    rows = ~np.isnan(want).all((1, 2))
    off = np.abs(got - want)[rows]
    assert (off <= bound(d, want, size)[rows]).all(), f"worst {off.max()} at {np.unravel_index(off.argmax(), off.shape)}"
    return got


IO = ["float32", "bfloat16"]
SHAPES = [(1, 1, 32), (4, 4, 64), (8, 2, 128), (14, 2, 64), (3, 1, 256), (64, 1, 32), (40, 2, 64)]


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (33, 4), (1000, 3)])
def test_decode_rows(device, io, heads, kv_heads, dim, window, sinks):
    d = make([(1, 1), (1, 5), (1, 33), (1, 100), (1, 257)], heads, kv_heads, dim, 16, io, seed=heads + dim)
    check(device, d, window, sinks, max_query_len=1)
    check(device, d, window, sinks)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 1), (24, 0), (64, 5)])
def test_prompt_chunks(device, io, heads, kv_heads, dim, window, sinks):
    check(device, make([(70, 70), (33, 150), (9, 9), (130, 131)], heads, kv_heads, dim, 16, io, seed=heads + dim), window, sinks)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("block", [1, 2, 3, 4, 8, 16, 20, 64, 200])
def test_mixed_batches_and_block_sizes(device, io, block):
    for dim in (64, 128):
        d = make([(1, 300), (45, 90), (1, 64), (3, 65), (1, 1), (2, 2), (80, 333), (1, 17)], 8, 2, dim, block, io, seed=block)
        for window, sinks in ((None, 0), (50, 0), (50, 7), (48, 8), (400, 0)):
            check(device, d, window, sinks)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (8, 2, 64), (4, 1, 32), (16, 2, 256)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (7, 2)])
def test_short_runs_that_share_a_tile(device, io, heads, kv_heads, dim, window, sinks):
    rng = np.random.default_rng(heads)
    for most in (4, 5, 9, 27):
        runs = [(n, n + int(rng.integers(0, 40))) for n in rng.integers(1, most + 1, 12).tolist() + [most] * 3]
        check(device, make(runs, heads, kv_heads, dim, 16, io, seed=most), window, sinks, max_query_len=most)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("block", [16, 48])
def test_whole_pages_beside_runs(device, io, dim, block):
    """Rows by themselves of every length around a page, beside runs; in some splits they have no key."""
    runs = [(1, n) for n in (1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 500)] + [(40, 60), (1, 0), (5, 300), (1, 129)]
    for splits in (0, 1, 5):
        check(device, make(runs, 6, 2, dim, block, io, seed=block + splits), num_splits=splits)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_splits_agree_with_the_definition(device, io, splits):
    d = make([(1, 700), (1, 3), (40, 500), (1, 129)], 8, 2, 128, 16, io, seed=splits)
    for window, sinks in ((None, 0), (1, 2), (90, 4)):
        check(device, d, window, sinks, num_splits=splits)


@pytest.mark.parametrize("io", IO)
def test_scales_of_every_block_and_head_count(device, io):
    """Scales far apart: a value read with another block's or head's would be off by powers of two."""
    d = make([(1, 200), (50, 170), (1, 90)], 6, 3, 64, 8, io, seed=5)
    rng = np.random.default_rng(2)
    # Far apart as values go, but the same for the scores of a head, whose weights would be one key's otherwise.
    d["vs"] = np.exp2(rng.integers(-60, 60, d["vs"].shape).astype(np.float64))
    d["v"] = np.where(np.abs(d["v"]) < 1, 1.0, d["v"])
    got = call(device, d).float().cpu().numpy().astype(np.float64)
    want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                                  d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    # Means of what differs by 2^120: relative to the largest value that the row sees with its weight.
    weighted, _ = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), np.abs(e4m3.values(d["v"], d["vs"])),
                                   d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    scores = (d["q"].shape[2] + 8) * 2.0**-24 * size[..., None]
    off = weighted * (2 * np.expm1(2 * scores) + (200 + 16) * 2.0**-24 + (2.0**-16 + 2.0**-8 if io == "bfloat16" else 0))
    assert (np.abs(got - want) <= off).all()


def test_rows_that_see_nothing_are_zeros(device):
    for io in IO:
        d = make([(1, 40), (1, 20), (30, 60)], 4, 2, 64, 16, io)
        d["positions"][0] = -1
        d["contexts"][1] = 0
        d["positions"][5:9] = -5  # rows of a run too
        for window, sinks in ((None, 0), (8, 2)):
            got = check(device, d, window, sinks)
            assert not got[0].any() and not got[1].any() and not got[5:9].any() and got[2].any()


@pytest.mark.parametrize("io", IO)
def test_rows_in_any_order_and_padding(device, io):
    import torch

    d = make([(20, 90), (1, 40), (30, 200)], 4, 2, 64, 16, io)
    order = np.random.default_rng(3).permutation(51)
    order = np.concatenate([order, np.arange(8, 20), np.arange(50, 20, -1)])
    d["q"], d["positions"], d["seqs"] = d["q"][order], d["positions"][order], d["seqs"][order]
    check(device, d, 25, 3)
    d["seqs"][10:14], d["seqs"][-1], d["seqs"][0] = -1, 3, 2**31 - 1
    for splits in (1, 4):
        out = torch.full(d["q"].shape, 5.0, dtype=d["q"].dtype, device=device)
        check(device, d, out=out, num_splits=splits)
        kept = out.float().cpu().numpy()
        assert (kept[10:14] == 5.0).all() and (kept[-1] == 5.0).all() and (kept[0] == 5.0).all()


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("block", [16, 6])
def test_bad_codes_and_scales_in_hidden_places_reach_no_output(device, io, block):
    """NaN codes, and scales that are no numbers, where no row looks."""
    d = make([(1, 100), (40, 100)], 4, 2, 64, block, io)
    clean = {w: call(device, d, *w).float().cpu() for w in ((None, 0), (24, 3))}
    unused = [b for b in range(d["k"].shape[0]) if b not in set(d["tables"][d["tables"] >= 0].tolist())]
    for name in ("k", "v"):
        d[name][unused] = np.nan
        d[name + "s"][unused] = np.nan
        for s in (0, 1):  # slots past a sequence's context
            d[name][d["tables"][s, 99 // block], 99 % block + 1 :] = np.nan
    for w, want in clean.items():
        assert (call(device, d, *w).float().cpu() == want).all()
    # Between the sinks and the first row's window.
    for s, hidden in ((0, (3, 40, 75)), (1, (3, 20, 36))):
        for j in hidden:
            for name in ("k", "v"):
                d[name][d["tables"][s, j // block], j % block] = np.nan
    assert (call(device, d, 24, 3).float().cpu() == clean[24, 3]).all()


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("splits", [1, 3])
def test_a_nan_reaches_the_rows_and_dimensions_that_see_it(device, io, splits):
    d = make([(1, 60), (20, 60)], 4, 2, 64, 16, io, seed=4)
    clean = call(device, d, num_splits=splits).float().cpu().numpy()
    want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                                  d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    off = bound(d, want, size)
    for s in (0, 1):
        d["v"][d["tables"][s, 3], 0, 1, 7] = np.nan  # key 48 of key head 1
    got = call(device, d, num_splits=splits).float().cpu().numpy()
    sees = d["positions"] >= 48
    assert np.isnan(got[sees][:, 2:, 7]).all()
    got[:, 2:, 7] = clean[:, 2:, 7]
    assert (np.abs(got - clean) <= 2 * off).all()


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [32, 128, 256])
@pytest.mark.parametrize("splits", [1, 4])
def test_nan_codes_of_every_head_dim(device, io, dim, splits):
    """Rows by themselves over whole pages and runs, in one call: hidden NaN codes reach nobody, seen ones those who see them."""
    d = make([(1, 60), (20, 60), (1, 200), (7, 33)], 6, 2, dim, 16, io, seed=dim)
    clean = call(device, d, num_splits=splits).float().cpu().numpy()
    for s, end in ((0, 60), (1, 60), (2, 200), (3, 33)):
        for name in ("k", "v"):
            d[name][d["tables"][s, end // 16], end % 16 :] = np.nan
    np.testing.assert_array_equal(call(device, d, num_splits=splits).float().cpu().numpy(), clean)
    for s in range(4):
        d["v"][d["tables"][s, 1], 9, 1, 5] = np.nan  # key 25 of key head 1
    got = call(device, d, num_splits=splits).float().cpu().numpy()
    sees = d["positions"] >= 25
    assert np.isnan(got[sees][:, 3:, 5]).all()
    want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), np.nan_to_num(e4m3.values(d["v"], d["vs"])),
                                  d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    off = bound(d, want, size)
    got[:, 3:, 5] = clean[:, 3:, 5]
    assert (np.abs(got - clean) <= 2 * off).all()


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("block", [16, 6])
@pytest.mark.parametrize("bad", [False, True])
def test_of_a_scale_its_exponent_alone_counts(device, io, block, bad):
    """Rows by themselves and runs, and both again where a NaN code has them computed by the definition: the same bits as with the
    scales' powers of two."""
    import torch

    d = make([(1, 60), (20, 60), (1, 200), (7, 33)], 6, 2, 64, block, io, seed=8)
    if bad:
        for s in range(4):
            d["v"][d["tables"][s, 25 // block], 25 % block, 1, 5] = np.nan
    clean = {w: call(device, d, *w).float().cpu() for w in ((None, 0), (24, 3))}
    rng = np.random.default_rng(3)
    for name in ("ks", "vs"):
        d[name] = d[name] * rng.choice([1.0, 1.25, 1.5, 1.9375, -1.0, -1.75], d[name].shape)
    for w, want in clean.items():
        got = call(device, d, *w).float().cpu()
        assert torch.equal(got.isnan(), want.isnan()) and bool(want.isnan().any()) == bad
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("block", [16, 6])
@pytest.mark.parametrize("name", ["ks", "vs"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_scales_that_are_no_numbers_are_nan_to_those_who_see_them(device, io, block, name, bad):
    d = make([(1, 60), (20, 60), (1, 200), (7, 33)], 6, 2, 64, block, io, seed=6)
    clean = call(device, d).float().cpu().numpy()
    for s in range(4):
        d[name][d["tables"][s, 25 // block], 1] = bad  # key head 1
    got = call(device, d).float().cpu().numpy()
    first = 25 // block * block  # of the block's keys
    sees = d["positions"] >= first
    assert np.isnan(got[sees][:, 3:]).all()
    np.testing.assert_array_equal(got[:, :3], clean[:, :3])
    np.testing.assert_array_equal(got[~sees], clean[~sees])


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("block", [16, 6])
@pytest.mark.parametrize("splits", [1, 3])
def test_large_queries_over_small_scales_beside_a_nan(device, io, block, splits):
    """Products of queries and codes pass float32's range, those of queries and keys do not: 2^120 * 2^8 * 8 against 2^31. A row's two
    largest scores lie 2^16 or more apart here and are off by at most (64 + 8) 2^-24 of their terms' sum, 2^29.5: less than 2^12. So
    each row is its largest key's value, in any type, and other dimensions' too where one is NaN."""
    d = make([(1, 60), (20, 60), (1, 200), (7, 33)], 6, 2, 64, block, io, seed=9)
    d["q"] = d["q"].sign() * 2.0**120
    d["ks"] = np.full(d["ks"].shape, 2.0**-100)
    clean = call(device, d, num_splits=splits).float().cpu().numpy()
    want, _ = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                               d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    np.testing.assert_array_equal(clean, want)
    for s in range(4):
        d["v"][d["tables"][s, 25 // block], 25 % block, 1, 5] = np.nan  # of key head 1
    got = call(device, d, num_splits=splits).float().cpu().numpy()
    assert np.isnan(got[d["positions"] >= 25][:, 3:, 5]).all()
    got[:, 3:, 5] = clean[:, 3:, 5]
    np.testing.assert_array_equal(got, clean)


def test_mixed_calls_captured_and_replayed_with_another_batch(device):
    """Tiles with shared runs, listed rows by pages, the order and the join in a graph whose lengths change between replays."""
    import torch

    from paged_kv_serving_amd import ops

    for io in IO:
        batches = [make([(n, n + more) for n, more in runs], 8, 2, 128, 16, io, seed=i) for i, runs in enumerate((
            [(9, 5), (1, 500), (1, 31), (27, 200), (1, 16), (25, 0)], [(1, 100), (30, 0), (1, 7), (1, 0), (21, 477), (10, 30)], [(10, 0)] * 6))]  # fmt: skip
        rows, blocks, width = 64, max(b["k"].shape[0] for b in batches), max(b["tables"].shape[1] for b in batches)

        def padded(d):
            n = d["seqs"].size
            pool = np.zeros((2, blocks, 16, 2, 128))
            scales = np.ones((2, blocks, 2), np.float32)
            for i, name in enumerate(("k", "v")):
                pool[i, : d[name].shape[0]], scales[i, : d[name].shape[0]] = d[name], d[name + "s"]
            tables = np.full((6, width), -1, np.int32)
            tables[:, : d["tables"].shape[1]] = d["tables"]
            q = torch.zeros((rows, 8, 128), dtype=d["q"].dtype)
            q[:n] = d["q"]
            return [q, torch.from_numpy(np.pad(d["positions"], (0, rows - n))), torch.from_numpy(np.pad(d["seqs"], (0, rows - n), constant_values=-1)),
                    codes_of(pool[0]), codes_of(pool[1]), *map(torch.from_numpy, scales), torch.from_numpy(tables), torch.from_numpy(d["contexts"])]  # fmt: skip

        assert all(b["seqs"].size <= rows for b in batches)
        held = [x.to(device) for x in padded(batches[0])]
        out = torch.zeros((rows, 8, 128), dtype=held[0].dtype, device=device)

        def run(result):
            return ops.paged_attention_e4m3(*held, 128**-0.5, max_context_len=512, max_query_len=30, out=result)

        run(out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(out)
        for d in batches + batches[::-1]:
            for a, b in zip(held, padded(d)):
                a.view(torch.uint8).copy_(b.view(torch.uint8)) if a.dtype == torch.float8_e4m3fn else a.copy_(b)
            out.fill_(7.0)
            graph.replay()
            eager = run(torch.full_like(out, 7.0))
            assert torch.equal(out, eager)
            n = d["seqs"].size
            assert (out[n:] == 7.0).all()  # padding is left as it was
            want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                                          d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
            assert (np.abs(out[:n].float().cpu().numpy().astype(np.float64) - want) <= bound(d, want, size)).all()


@pytest.mark.parametrize("io", IO)
def test_blocks_outside_the_pool_are_skipped(device, io):
    d = make([(1, 100), (40, 100), (1, 20)], 4, 2, 64, 16, io)
    d["tables"][0, 3], d["tables"][1, 2], d["tables"][1, 5], d["tables"][2, :2] = -1, 10**6, -5, 2**31 - 1
    for window, sinks, splits in ((None, 0, 1), (None, 0, 3), (60, 3, 1), (60, 3, 3)):
        got = check(device, d, window, sinks, num_splits=splits)
        assert not got[-1].any()  # nothing left to see


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales_of_the_scores(device, io, scale):
    d = make([(1, 120), (40, 120)], 4, 2, 64, 16, io)
    d["scale"] = scale
    if scale == 40.0:
        assert np.isfinite(call(device, d).float().cpu().numpy()).all()
    else:
        check(device, d)


@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("io", IO)
def test_many_rows_and_rows_beside_runs(device, io, splits):
    """More workgroups than CUs (two key heads to a workgroup), and rows beside a run that share a few."""
    runs = [(1, 5 + 7 * i % 90) for i in range(180)]
    check(device, make(runs, 8, 8, 64, 16, io, seed=11), num_splits=splits)
    check(device, make(runs[:100], 14, 7, 128, 16, io, seed=11), num_splits=splits, max_query_len=1)
    check(device, make(runs[:70], 16, 16, 256, 16, io, seed=11), num_splits=splits, max_query_len=1)
    runs[60:60] = [(30, 130)]
    check(device, make(runs, 8, 8, 64, 16, io, seed=12), 40, 2, num_splits=splits)


def test_attention_past_32_bit_offsets(device):
    import torch

    from paged_kv_serving_amd import ops

    heads, dim, block = 8, 128, 16
    blocks = (1 << 32) // (heads * dim * block) + 64
    k, v = (torch.zeros((blocks, block, heads, dim), dtype=torch.uint8, device=device) for _ in range(2))
    ks, vs = (torch.zeros((blocks, heads), device=device) for _ in range(2))
    d = make([(1, 100), (30, 90)], 16, heads, dim, block, "bfloat16")
    used = d["k"].shape[0]
    for pool, scales, name in ((k, ks, "k"), (v, vs, "v")):
        pool[-used:], scales[-used:] = codes_of(d[name]).view(torch.uint8).to(device), torch.from_numpy(d[name + "s"].astype(np.float32)).to(device)
    want = call(device, d)
    tables = torch.from_numpy(np.where(d["tables"] >= 0, d["tables"] + blocks - used, -1).astype(np.int32)).to(device)
    put = lambda x: torch.from_numpy(x).to(device)  # noqa: E731
    got = ops.paged_attention_e4m3(d["q"].to(device), put(d["positions"]), put(d["seqs"]), k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs,
                                   tables, put(d["contexts"]), d["scale"], max_context_len=100)  # fmt: skip
    assert torch.equal(got, want)


def test_twice_the_same_bits_and_two_streams(device):
    import torch

    batches = [make([(1, 800), (60, 500)], 8, 2, 64, 16, "bfloat16", seed=s) for s in (1, 2)]
    want = [call(device, d, num_splits=4) for d in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for d, stream in zip(batches, streams):
        with torch.cuda.stream(stream):
            got.append(call(device, d, num_splits=4))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_no_rows_no_context_no_blocks_and_refusals(device):
    import torch

    d = make([(1, 20), (3, 30)], 4, 2, 64, 16, "float32")
    empty = {**d, "q": d["q"][:0], "positions": d["positions"][:0], "seqs": d["seqs"][:0]}
    assert call(device, empty).shape == (0, 4, 64)
    assert not call(device, {**d, "contexts": np.zeros(2, np.int32)}, max_context_len=0).any()
    bad = [
        ({}, {"window": 0}), ({}, {"sinks": 1}), ({}, {"window": 4, "sinks": -1}), ({}, {"num_splits": 65}), ({}, {"max_context_len": 10_000}),
        ({}, {"out": torch.zeros((4, 4, 64), device=device, dtype=torch.bfloat16)}), ({}, {"num_splits": 2, "workspace": torch.zeros(4, device=device)}),
        ({"q": d["q"].half()}, {}), ({"q": d["q"][:, :3]}, {}), ({"ks": d["ks"][:1]}, {}), ({"vs": d["vs"].T.copy()}, {}), ({"v": d["v"][:1]}, {}),
        ({"seqs": d["seqs"].astype(np.int64)}, {}), ({"tables": d["tables"].astype(np.int64)}, {}), ({"contexts": d["contexts"][:1]}, {}),
        ({"k": d["k"][0], "v": d["v"][0]}, {}),
    ]  # fmt: skip
    for change, more in bad:
        with pytest.raises(ValueError):
            call(device, {**d, **change}, **more)


# --- decode rows in equal shares -------------------------------------------------------------------

UNEVEN = [700, 1, 33, 2000, 64, 32, 5, 900, 16, 1200, 31, 300, 2, 17, 450, 100]  # together more than one workgroup's share


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 128), (8, 8, 64), (12, 6, 128), (4, 4, 32), (3, 3, 128), (4, 2, 256), (40, 2, 64), (64, 4, 32)])
def test_rows_in_equal_shares(device, io, heads, kv_heads, dim):
    """Rows in one share, in several, and shares of several rows; four, two or one key head to a workgroup."""
    runs = [(1, c) for c in UNEVEN * 2]
    check(device, make(runs, heads, kv_heads, dim, 16, io, seed=heads + dim), max_query_len=1)


@pytest.mark.parametrize("block", [16, 32, 48, 1024])
def test_shares_of_other_blocks(device, block):
    check(device, make([(1, c) for c in UNEVEN * 2], 8, 4, 64, block, "bfloat16", seed=block), max_query_len=1)


@pytest.mark.parametrize("io", IO)
def test_shares_with_rows_that_see_nothing_padding_and_missing_blocks(device, io):
    import torch

    d = make([(1, c) for c in UNEVEN * 2], 8, 4, 64, 16, io, seed=3)
    d["contexts"][[0, 5, 6, 31]] = 0
    d["positions"][9] = -1
    d["positions"][20] = 100  # fewer keys than its context
    d["seqs"][[3, 14, 30]] = -1, 32, 2**31 - 1
    d["tables"][7, 10:20], d["tables"][19, 0], d["tables"][25, -5:] = -1, 10**6, -2
    out = torch.full(d["q"].shape, 5.0, dtype=d["q"].dtype, device=device)
    got = check(device, d, max_query_len=1, out=out)
    assert not got[[0, 5, 6, 9, 31]].any() and (got[[3, 14, 30]] == 5.0).all()
    d["contexts"][:] = 0
    assert not call(device, d, max_query_len=1, max_context_len=2000).float().cpu().numpy()[[0, 1, 2]].any()


@pytest.mark.parametrize("io", IO)
def test_shares_with_nan_codes(device, io):
    d = make([(1, c) for c in UNEVEN * 2], 8, 4, 64, 16, io, seed=4)
    clean = check(device, d, max_query_len=1)
    want, size = window_attention(d["q"].float().numpy(), d["positions"], d["seqs"], e4m3.values(d["k"], d["ks"]), e4m3.values(d["v"], d["vs"]),
                                  d["tables"], d["contexts"], d["scale"], CAUSAL, 0)  # fmt: skip
    off = bound(d, want, size)
    for s, j, h, dim in ((3, 1999, 1, 7), (7, 0, 2, 63), (0, 350, 0, 0), (1, 0, 3, 5)):
        d["v"][d["tables"][s, j // 16], j % 16, h, dim] = np.nan
    got = call(device, d, max_query_len=1).float().cpu().numpy()
    for s, h, dim in ((3, 1, 7), (7, 2, 63), (0, 0, 0), (1, 3, 5)):
        assert np.isnan(got[s, 2 * h : 2 * h + 2, dim]).all()
        got[s, 2 * h : 2 * h + 2, dim] = clean[s, 2 * h : 2 * h + 2, dim]
    assert (np.abs(got - clean) <= 2 * off).all()


@pytest.mark.parametrize("rows", [1, 2, 1023, 1024, 1025])
def test_as_many_rows_as_shares_take_and_more(device, rows):
    d = make([(1, 40 if rows > 2 else 33000)] * rows, 4, 4, 32, 16, "bfloat16", seed=rows)
    rng = np.random.default_rng(rows)
    if rows > 2:
        d["contexts"] = rng.integers(0, 41, rows).astype(np.int32)
        d["positions"] = (d["contexts"] - 1).astype(np.int32)
    check(device, d, max_query_len=1, max_context_len=int(max(40, d["contexts"].max())))


def test_shares_captured_and_replayed_with_another_batch(device):
    """One graph and one workspace, batches whose rows and lengths change."""
    import torch

    from paged_kv_serving_amd import ops

    most, heads, kv_heads, dim = 2000, 8, 4, 64
    rng = np.random.default_rng(1)
    cases = [make([(1, int(c)) for c in lengths], heads, kv_heads, dim, 16, "bfloat16", seed=i)
             for i, lengths in enumerate((UNEVEN * 2, [2000] * 32, rng.integers(1, 2001, 32), [1] * 31 + [1990]))]  # fmt: skip
    blocks, width = max(c["k"].shape[0] for c in cases), most // 16
    buf = {
        "q": torch.zeros((32, heads, dim), dtype=torch.bfloat16, device=device), "tables": torch.zeros((32, width), dtype=torch.int32, device=device),
        **{name: torch.zeros((blocks, 16, kv_heads, dim), dtype=torch.uint8, device=device) for name in "kv"},
        **{name: torch.ones((blocks, kv_heads), device=device) for name in ("ks", "vs")},
        **{name: torch.zeros(32, dtype=torch.int32, device=device) for name in ("positions", "seqs", "contexts")},
    }  # fmt: skip
    out = torch.zeros_like(buf["q"])
    need = ops.e4m3_workspace_bytes(32, heads, kv_heads, dim, block_size=16, max_context_len=most, max_query_len=1)
    workspace = torch.full((need // 4,), float("nan"), device=device)

    def run():
        ops.paged_attention_e4m3(buf["q"], buf["positions"], buf["seqs"], buf["k"].view(torch.float8_e4m3fn), buf["v"].view(torch.float8_e4m3fn), buf["ks"],
                                 buf["vs"], buf["tables"], buf["contexts"], dim**-0.5, max_context_len=most, max_query_len=1, out=out, workspace=workspace)  # fmt: skip

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for d in cases * 2:
        for name in "kv":
            buf[name][: d[name].shape[0]].copy_(codes_of(d[name]).view(torch.uint8))
            buf[name + "s"][: d[name].shape[0]].copy_(torch.from_numpy(d[name + "s"]))
        buf["q"].copy_(d["q"])
        for name in ("positions", "seqs", "contexts"):
            buf[name].copy_(torch.from_numpy(d[name]))
        buf["tables"].zero_()
        cols = min(width, d["tables"].shape[1])
        buf["tables"][:, :cols].copy_(torch.from_numpy(d["tables"][:, :cols]))
        graph.replay()
        torch.cuda.synchronize()
        wide = {**d, "tables": np.pad(d["tables"], ((0, 0), (0, max(0, width - d["tables"].shape[1]))), constant_values=-7)}
        assert torch.equal(out, call(device, wide, max_query_len=1, max_context_len=most))


def test_the_workspace_that_a_call_needs(device):
    import torch

    from paged_kv_serving_amd import ops

    d = make([(1, c) for c in UNEVEN * 2], 8, 4, 64, 16, "bfloat16", seed=3)
    need = ops.e4m3_workspace_bytes(32, 8, 4, 64, block_size=16, max_context_len=2000, max_query_len=1)
    assert need > 0
    check(device, d, max_query_len=1, workspace=torch.empty(need // 4, device=device))
    with pytest.raises(ValueError, match="workspace"):
        call(device, d, max_query_len=1, workspace=torch.empty(need // 4 - 1, device=device))
    for more in ({"num_splits": 3}, {"window": 100}, {"max_query_len": 40}, {}):
        for block in (16, 12):
            e = make([(1, 700), (1, 5)], 4, 4, 64, block, "float32", seed=1)
            need = ops.e4m3_workspace_bytes(2, 4, 4, 64, block_size=block, max_context_len=700, **more)
            check(device, e, workspace=torch.empty(max(1, need // 4), device=device), **more)
