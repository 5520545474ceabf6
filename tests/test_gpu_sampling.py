"""sample_tokens against the float64 definition, at the sizes, settings and logits where it can go wrong."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu


def draw(device, logits, uniforms, **settings):
    """Tokens of float32 or bfloat16 ``logits`` (a torch CPU tensor)."""
    import torch

    from paged_kv_serving_amd import ops

    put = {k: torch.as_tensor(v).to(device) if isinstance(v, np.ndarray) else v for k, v in settings.items()}
    u = torch.as_tensor(np.asarray(uniforms, np.float32)).to(device)
    return ops.sample_tokens(logits.to(device), u, **put).cpu().numpy()


def expect(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]
    each = [np.broadcast_to(np.asarray(v), rows) for v in (temperature, top_k, top_p, min_p)]
    data = logits.float().numpy()
    return np.asarray([sample_row(data[r], uniforms[r], *(e[r].item() for e in each)) for r in range(rows)])


def make(rows, vocab, seed, spread=2.0, dtype="float32"):
    import torch

    rng = np.random.default_rng(seed)
    logits = torch.from_numpy((spread * rng.standard_normal((rows, vocab))).astype(np.float32))
    return logits.to(getattr(torch, dtype)), rng.random(rows, dtype=np.float32)


SETTINGS = [
    {},
    {"temperature": 0.7},
    {"top_k": 1},
    {"top_k": 20},
    {"top_k": 700, "temperature": 1.3},
    {"top_k": 3000},
    {"top_p": 0.9},
    {"top_p": 0.05},
    {"min_p": 0.1},
    {"min_p": 1.0},
    {"top_k": 50, "top_p": 0.9, "min_p": 0.02, "temperature": 0.8},
    {"temperature": 0.0},
    {"temperature": 1e-3},
    {"temperature": 1e6},
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 255, 1000, 4097, 50257])
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
def test_rows_match_the_definition(device, settings, vocab, dtype):
    logits, u = make(5, vocab, vocab + len(settings), dtype=dtype)
    np.testing.assert_array_equal(draw(device, logits, u, **settings), expect(logits, u, **settings))


@pytest.mark.parametrize("spread", [0.0, 1e-6, 0.01, 30.0, 1e20])
@pytest.mark.parametrize("settings", [{}, {"top_k": 900}, {"top_p": 0.6}, {"top_k": 5000, "top_p": 0.5}], ids=str)
def test_narrow_and_wide_rows(device, settings, spread):
    logits, u = make(4, 20011, 3, spread=spread)
    np.testing.assert_array_equal(draw(device, logits, u, **settings), expect(logits, u, **settings))


def test_settings_of_each_row(device):
    rows, vocab = 64, 9001
    logits, u = make(rows, vocab, 11)
    rng = np.random.default_rng(12)
    settings = {
        "temperature": rng.choice(np.asarray([0.0, 0.5, 1.0, 2.0], np.float32), rows),
        "top_k": rng.choice(np.asarray([0, 1, 3, 40, 1000, 9001, 20000], np.int32), rows),
        "top_p": rng.choice(np.asarray([1.0, 0.1, 0.9, 0.99], np.float32), rows),
        "min_p": rng.choice(np.asarray([0.0, 0.05, 0.5], np.float32), rows),
    }
    np.testing.assert_array_equal(draw(device, logits, u, **settings), expect(logits, u, **settings))


@pytest.mark.parametrize("vocab", [4, 1024, 5000, 131072])
def test_equal_logits_go_by_their_ids(device, vocab):
    import torch

    u = np.asarray([0.0, 0.25, 0.5, 0.75, 0.999], np.float32)
    logits = torch.full((5, vocab), -3.25)
    got = draw(device, logits, u)
    np.testing.assert_array_equal(got, np.floor(u.astype(np.float64) * vocab))
    got = draw(device, logits, u, top_k=2, top_p=0.5)  # the first of two equal tokens has half their mass
    np.testing.assert_array_equal(got, 0)
    half = draw(device, logits, u, top_p=0.5)
    np.testing.assert_array_equal(half, np.floor(u.astype(np.float64) * (vocab // 2)))


def test_signed_zeros_tie(device):
    import torch

    logits = torch.tensor([[-0.0, 0.0, -0.0, 0.0]]).repeat(4, 1)
    np.testing.assert_array_equal(draw(device, logits, [0.1, 0.3, 0.6, 0.9]), [0, 1, 2, 3])


def test_many_ties_across_a_bin(device):
    """More equal tokens than any list holds, above and below others, cut by count and by mass."""
    import torch

    rng = np.random.default_rng(5)
    values = rng.choice(np.asarray([0.0, 0.5, 0.50000006, 1.0], np.float32), (6, 60000), p=[0.3, 0.3, 0.3, 0.1])
    logits, u = torch.from_numpy(values), rng.random(6, dtype=np.float32)
    for settings in ({}, {"top_k": 20000}, {"top_p": 0.7}, {"top_k": 30001, "top_p": 0.95}):
        np.testing.assert_array_equal(draw(device, logits, u, **settings), expect(logits, u, **settings))


def test_outlier_above_a_narrow_bulk(device):
    """One token far above tens of thousands in a range of 1e-4: they share a few bins."""
    import torch

    rng = np.random.default_rng(6)
    values = (1e-4 * rng.standard_normal((4, 70001))).astype(np.float32)
    values[:, 4321] = 9.0
    logits, u = torch.from_numpy(values), np.asarray([0.05, 0.2, 0.6, 0.99], np.float32)
    for settings in ({}, {"top_k": 40000}, {"top_p": 0.5}):
        np.testing.assert_array_equal(draw(device, logits, u, **settings), expect(logits, u, **settings))


def test_rows_with_infinities_and_nan(device):
    import torch

    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([
        [-inf, 1.0, -inf, 1.0],  # masked tokens are never drawn
        [-inf, -inf, -inf, -inf],  # nothing left: the greedy token
        [0.0, inf, 5.0, inf],  # +inf share the mass
        [0.0, nan, 9.0, nan],  # the first NaN
        [-3.4e38, -inf, -3.4e38, -inf],  # the type's lowest value is a number
        [-inf, -inf, 2.0, -inf],
        [3.0e38, -3.0e38, 3.0e38, 0.0],
    ])  # fmt: skip
    for settings in ({}, {"top_k": 2}, {"top_p": 0.9}, {"min_p": 0.5}, {"temperature": 0.0}, {"temperature": float("inf")}):
        for u in (0.0, 0.3, 0.8):
            us = np.full(7, u, np.float32)
            np.testing.assert_array_equal(draw(device, logits, us, **settings), expect(logits, us, **settings), err_msg=str((settings, u)))


def test_uniforms_outside_their_range_stay_in_the_row(device):
    logits, _ = make(4, 5000, 21)
    u = np.asarray([-1.0, np.nan, 1.0, 5.0], np.float32)
    got = draw(device, logits, u, top_k=10)
    order = np.argsort(-logits.numpy(), axis=1, kind="stable")
    np.testing.assert_array_equal(got, [order[0, 0], order[1, 0], order[2, 9], order[3, 9]])


def test_settings_outside_their_range(device):
    """Per-row settings are not read on the host: each has a meaning."""
    logits, _ = make(4, 3000, 22)
    order = np.argsort(-logits.numpy(), axis=1, kind="stable")
    u = np.full(4, 0.999, np.float32)
    got = draw(device, logits, u, top_p=np.asarray([0.0, -1.0, np.nan, 1e-30], np.float32))
    np.testing.assert_array_equal(got, order[:, 0])
    got = draw(device, logits, u, min_p=np.asarray([1.5, np.inf, 1.0, 2.0], np.float32))
    np.testing.assert_array_equal(got, order[:, 0])
    got = draw(device, logits, u, temperature=np.asarray([-1.0, np.nan, 0.0, -0.0], np.float32))
    np.testing.assert_array_equal(got, order[:, 0])
    got = draw(device, logits, u, top_k=np.asarray([-5, 0, 3000, 2**31 - 1], np.int32), min_p=np.asarray([-1.0, np.nan, 0.0, 0.0], np.float32))
    np.testing.assert_array_equal(got, expect(logits, u))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_rows_and_odd_starts(device, dtype):
    import torch

    from paged_kv_serving_amd import ops

    wide, u = make(9, 3333, 31, dtype=dtype)
    want_all = wide[1:8, 3:3001]
    data = wide.to(device)
    got = ops.sample_tokens(data[1:8, 3:3001], torch.from_numpy(u[:7]).to(device), top_p=0.8)
    np.testing.assert_array_equal(got.cpu().numpy(), expect(want_all, u[:7], top_p=0.8))
    turned = data.t().contiguous().t()  # columns apart
    got = ops.sample_tokens(turned, torch.from_numpy(u).to(device), top_k=30)
    np.testing.assert_array_equal(got.cpu().numpy(), expect(wide, u, top_k=30))


def test_empty_batch_and_output_buffer(device):
    import torch

    from paged_kv_serving_amd import ops

    empty = ops.sample_tokens(torch.zeros((0, 10), device=device), torch.zeros(0, device=device))
    assert empty.shape == (0,) and empty.dtype == torch.int32
    logits, u = make(3, 100, 41)
    out = torch.full((3,), -1, dtype=torch.int32, device=device)
    assert ops.sample_tokens(logits.to(device), torch.from_numpy(u).to(device), out=out) is out
    np.testing.assert_array_equal(out.cpu().numpy(), expect(logits, u))


def test_a_token_does_not_depend_on_its_batch(device):
    logits, u = make(40, 30000, 51)
    together = draw(device, logits, u, top_p=0.95, top_k=500)
    alone = [draw(device, logits[r : r + 1], u[r : r + 1], top_p=0.95, top_k=500)[0] for r in range(40)]
    np.testing.assert_array_equal(together, alone)


def test_shares_of_a_large_sample(device):
    """Drawn shares of a known distribution, and the draw's order: growing uniforms fall through the ranks."""
    import torch

    p = np.asarray([0.5, 0.25, 0.125, 0.125])
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)  # evenly spread: every share is exact to one draw
    logits = torch.from_numpy(np.log(p).astype(np.float32)).repeat(n, 1)
    got = draw(device, logits, u)
    assert (np.diff(got) >= 0).all()
    assert np.abs(np.bincount(got, minlength=4) - n * p).max() <= 1


def test_captured_and_replayed(device):
    import torch

    from paged_kv_serving_amd import ops

    logits = torch.zeros((6, 20000), device=device)
    u = torch.zeros(6, device=device)
    out = torch.zeros(6, dtype=torch.int32, device=device)
    ops.sample_tokens(logits, u, top_p=0.9, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_tokens(logits, u, top_p=0.9, top_k=300, out=out)
    for seed in range(4):
        data, us = make(6, 20000, 60 + seed)
        logits.copy_(data)
        u.copy_(torch.from_numpy(us))
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(out.cpu().numpy(), expect(data, us, top_p=0.9, top_k=300))


def test_on_a_stream_of_its_own(device):
    import torch

    from paged_kv_serving_amd import ops

    data, us = make(8, 30000, 71)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.sample_tokens(data.to(device), torch.from_numpy(us).to(device), min_p=0.02)
    stream.synchronize()
    np.testing.assert_array_equal(got.cpu().numpy(), expect(data, us, min_p=0.02))


def test_refusals(device):
    import torch

    from paged_kv_serving_amd import ops

    x = torch.zeros((2, 8), device=device)
    u = torch.zeros(2, device=device)
    for bad in (
        {"temperature": -1.0}, {"temperature": float("nan")}, {"top_k": -1}, {"top_p": 0.0}, {"top_p": 1.5}, {"min_p": -0.1}, {"min_p": 1.1},
        {"temperature": torch.ones(3, device=device)}, {"top_k": torch.ones(2, device=device)}, {"top_p": torch.ones(2)},
        {"out": torch.zeros(2, device=device)}, {"out": torch.zeros(2, dtype=torch.int32)},
    ):  # fmt: skip
        with pytest.raises(ValueError):
            ops.sample_tokens(x, u, **bad)
    for logits, uniforms in ((x.half(), u), (x[0], u), (x, u[:1]), (x, u.double()), (x[:, :0], u), (x.cpu(), u), (x, u.cpu())):
        with pytest.raises(ValueError):
            ops.sample_tokens(logits, uniforms)


def test_one_row_expanded_over_the_batch(device):
    logits, _ = make(1, 300, 8)
    uniforms = np.linspace(0, 0.99, 7, dtype=np.float32)
    assert draw(device, logits.to(device).expand(7, 300), uniforms).tolist() == expect(logits.expand(7, 300), uniforms).tolist()


@pytest.mark.parametrize("spread", [0.3, 1.0, 3.0, 12.0])
@pytest.mark.parametrize("more", [{}, {"top_k": 6000}, {"min_p": 1e-4}], ids=str)
def test_the_nucleus_end_and_the_draw_wherever_they_lie(device, more, spread):
    """From the draw in front of everything to the draw of the nucleus's last token."""
    settings = [(u, p) for u in (0.0, 0.02, 0.5, 0.97, np.nextafter(np.float32(1), np.float32(0))) for p in (0.02, 0.5, 0.9, 0.9999)]
    logits, _ = make(len(settings), 20011, 77, spread)
    uniforms = np.asarray([u for u, _ in settings], np.float32)
    more = {**more, "top_p": np.asarray([p for _, p in settings], np.float32)}
    assert draw(device, logits, uniforms, **more).tolist() == expect(logits, uniforms, **more).tolist()
