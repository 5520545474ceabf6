"""What pkv_rope_append_axes, pkv_window_attention and pkv_sample_tokens refuse, and the window's host
functions, at the C ABI: every refusal returns before any HIP call, so no GPU is needed and the
pointers are made up. (A call whose arguments are all right would go on to the device; none is made.)"""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from paged_kv_serving_amd import _native

HEADER = (Path(__file__).resolve().parents[1] / "include" / "pkv.h").read_text()
EINVAL, EUNSUPPORTED, FAKE = -1, -2, 0x10000


def structure(name: str):
    """A ctypes structure with the fields that the header declares."""
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, HEADER, re.S).group(1)
    fields = []
    for kind, star, field, count in re.findall(r"(?:const )?(\w+)(\*?) (\w+)(?:\[(\w+)\])?;", body):
        c_type = ctypes.c_void_p if star else getattr(ctypes, {"float": "c_float"}.get(kind, "c_" + kind[:-2]))
        fields.append((field, c_type * 4 if count == "PKV_MAX_ROPE_AXES" else c_type))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        _native.build()
    return _native.library()


def refused(function, kind, good: dict, **changes) -> int:
    args = kind()
    for name, value in {**good, **changes}.items():
        setattr(args, name, tuple(value) if isinstance(value, (tuple, list)) else value)
    return function(ctypes.addressof(args), 0, None)


ROPE = dict(
    rotated_queries=FAKE, queries=2 * FAKE, keys=3 * FAKE, values=4 * FAKE, rotated_token_stride=256, query_token_stride=256,
    key_token_stride=128, value_token_stride=128, positions=5 * FAKE, position_axis_stride=9, cos_table=6 * FAKE,
    sin_table=7 * FAKE, table_rows=64, key_pool=8 * FAKE, value_pool=9 * FAKE, num_slots=80, slot_mapping=10 * FAKE,
    num_tokens=9, io_dtype=0, pool_dtype=0, num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=48, num_axes=3,
    interleaved=0, sections=(8, 8, 8, 0),
)  # fmt: skip
WINDOW = dict(
    out=FAKE, queries=2 * FAKE, query_token_stride=512, query_positions=3 * FAKE, query_seq=4 * FAKE, num_queries=7,
    key_cache=5 * FAKE, value_cache=6 * FAKE, num_blocks=40, block_tables=7 * FAKE, context_lens=8 * FAKE, workspace=9 * FAKE,
    workspace_bytes=1 << 20, q_dtype=0, kv_dtype=0, block_size=16, block_table_stride=10, num_seqs=4, num_heads=8,
    num_kv_heads=2, head_dim=64, window=32, sinks=2, max_context_len=160, max_query_len=7, num_splits=2, scale=0.125,
)  # fmt: skip
SAMPLE = dict(token_ids=FAKE, logits=2 * FAKE, row_stride=100, num_rows=3, vocab_size=100, uniforms=3 * FAKE, dtype=0,
              temperature=1.0, top_p=1.0)  # fmt: skip


@pytest.mark.parametrize("changes", [
    {"num_tokens": -1}, {"num_heads": 0}, {"num_kv_heads": 0}, {"head_dim": 1}, {"rotary_dim": 0}, {"rotary_dim": 47},
    {"rotary_dim": 66}, {"num_slots": -1}, {"table_rows": -1}, {"io_dtype": 2}, {"pool_dtype": 7}, {"num_axes": 0},
    {"num_axes": 5}, {"sections": (8, 8, 7, 0)}, {"sections": (8, -8, 24, 0)}, {"sections": (8, 8, 8, 0), "num_axes": 2},
    {"sections": (6, 9, 9, 0), "interleaved": 1}, {"query_token_stride": 255}, {"rotated_token_stride": 255},
    {"key_token_stride": 127}, {"value_token_stride": 0}, {"position_axis_stride": -1}, {"queries": None}, {"keys": None},
    {"values": None}, {"rotated_queries": None}, {"positions": None}, {"cos_table": None}, {"sin_table": None},
    {"key_pool": None}, {"value_pool": None}, {"slot_mapping": None},
    {"rotated_queries": 2 * FAKE, "rotated_token_stride": 512},
], ids=str)  # fmt: skip
def test_rope_refusals(lib, changes) -> None:
    assert refused(lib.pkv_rope_append_axes, structure("pkv_rope_axes"), ROPE, **changes) == EINVAL


@pytest.mark.parametrize("changes,code", [
    *(({name: -1}, EINVAL) for name in ("num_queries", "num_seqs", "num_blocks", "block_table_stride", "sinks",
                                        "max_context_len", "max_query_len", "num_splits")),
    *(({name: 0}, EINVAL) for name in ("num_heads", "num_kv_heads", "block_size", "window")),
    *(({name: None}, EINVAL) for name in ("out", "queries", "query_positions", "query_seq", "key_cache", "value_cache",
                                          "block_tables", "context_lens", "workspace")),
    *(({name: FAKE + 8}, EINVAL) for name in ("out", "queries", "key_cache", "value_cache", "workspace")),
    ({"num_heads": 7}, EINVAL), ({"num_splits": 65}, EINVAL), ({"max_context_len": 161}, EINVAL),
    ({"q_dtype": 2}, EINVAL), ({"kv_dtype": -1}, EINVAL), ({"q_dtype": 1}, EUNSUPPORTED),
    ({"head_dim": 48}, EUNSUPPORTED), ({"head_dim": 512}, EUNSUPPORTED), ({"num_heads": 130}, EUNSUPPORTED),
    ({"num_blocks": 1 << 27}, EUNSUPPORTED), ({"num_blocks": 1 << 62}, EUNSUPPORTED),
    ({"max_context_len": (1 << 30) + 1, "block_table_stride": 1 << 30}, EUNSUPPORTED),
    ({"query_token_stride": 511}, EINVAL), ({"query_token_stride": 514}, EINVAL), ({"workspace_bytes": 100}, EINVAL),
], ids=str)  # fmt: skip
def test_window_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_window_attention, structure("pkv_window"), WINDOW, **changes) == code


@pytest.mark.parametrize("changes,code", [
    ({"num_rows": -1}, EINVAL), ({"vocab_size": 0}, EINVAL), ({"vocab_size": 1 << 31, "row_stride": 1 << 31}, EINVAL),
    ({"row_stride": 99}, EINVAL), ({"dtype": 2}, EINVAL), ({"token_ids": None}, EINVAL), ({"logits": None}, EINVAL),
    ({"uniforms": None}, EINVAL), ({"num_rows": 1 << 31}, EUNSUPPORTED), ({"num_rows": 1 << 22}, EUNSUPPORTED),
], ids=str)  # fmt: skip
def test_sampling_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_sample_tokens, structure("pkv_sample"), SAMPLE, **changes) == code


def test_no_arguments_and_nothing_to_do(lib) -> None:
    for function in (lib.pkv_rope_append_axes, lib.pkv_window_attention, lib.pkv_sample_tokens):
        assert function(None, 0, None) == EINVAL
    assert refused(lib.pkv_rope_append_axes, structure("pkv_rope_axes"), ROPE, num_tokens=0) == 0
    assert refused(lib.pkv_window_attention, structure("pkv_window"), WINDOW, num_queries=0) == 0
    assert refused(lib.pkv_sample_tokens, structure("pkv_sample"), SAMPLE, num_rows=0) == 0


def test_window_workspace_holds_every_split_and_the_row_list(lib) -> None:
    size = lib.pkv_window_workspace_bytes
    assert size(64, 32, 128, 1, 1) == 0
    assert size(64, 32, 128, 1, 8) == 64 * 32 * 8 * 130 * 4
    assert size(3, 1, 32, 1, 3) == (3 * 3 * 34 * 4 + 15) // 16 * 16  # maxima and sums end on 16 bytes, then the outputs
    assert size(3, 1, 32, 1, 3) >= ((2 * 9 + 3) // 4 * 4 + 9 * 32) * 4
    assert size(64, 32, 128, 64, 1) >= (64 + 1) * 4  # a counter and a row each
    for bad in ((-1, 1, 32, 1, 1), (1, 0, 32, 1, 1), (1, 1, 0, 1, 1), (1, 1, 32, -1, 1), (1, 1, 32, 1, 0), (1, 1, 32, 1, 65)):
        assert size(*bad) == EINVAL


def test_window_splits_follow_the_work(lib) -> None:
    splits = lib.pkv_window_splits  # queries, heads, kv_heads, window, sinks, context, rows of a run
    assert splits(1, 64, 8, 4096, 4, 32768, 1) == 16  # few rows: 256 keys to a split
    assert splits(1, 64, 8, 1000, 4, 32768, 1) == 1  # but few keys are not split
    assert splits(256, 64, 8, 4096, 4, 32768, 1) == 1  # enough rows
    assert splits(36, 64, 8, 4096, 4, 32768, 1) == 4  # 288 workgroups would leave 224 of 512 places idle
    assert splits(36, 64, 8, 2048, 0, 32768, 1) == 2 and splits(36, 64, 8, 512, 0, 32768, 1) == 1
    assert splits(1, 64, 8, 100, 0, 32768, 1) == splits(1, 64, 8, 4096, 4, 100, 1) == 1  # few keys
    assert splits(1, 1, 1, 1 << 20, 0, 1 << 20, 1) == 64  # no more than the most
    assert splits(512, 8, 8, 4096, 0, 4096, 512) > splits(8192, 8, 8, 4096, 0, 4096, 512) >= 1
    assert splits(0, 8, 8, 16, 0, 0, 0) >= 1
    for bad in ((-1, 8, 8, 1, 0, 1, 1), (1, 8, 0, 1, 0, 1, 1), (1, 7, 2, 1, 0, 1, 1), (1, 8, 8, 0, 0, 1, 1),
                (1, 8, 8, 1, -1, 1, 1), (1, 8, 8, 1, 0, -1, 1), (1, 8, 8, 1, 0, 1, -1), (1, 65, 1, 1, 0, 1, 1)):  # fmt: skip
        assert splits(*bad) == EINVAL


def test_tensors_off_the_device_are_refused_by_name(lib) -> None:
    import torch

    from paged_kv_serving_amd import ops

    f, i32, i64 = torch.zeros(1, 2, 32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    pool, table = torch.zeros(4, 8, 2, 32), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        ops.rope_append_axes(pool, pool, f, f, f, i64, torch.zeros(4, 16), torch.zeros(4, 16), i64)
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_attention_window(f, i32, i32, pool, pool, table, i32, 1.0, window=4, max_context_len=8)
    with pytest.raises(ValueError, match="HIP device"):
        ops.sample_tokens(torch.zeros(1, 9), torch.zeros(1))
    host = _native.bound_host()
    assert host.one_device(f, i32) == host.one_device() == -1
    with pytest.raises(AttributeError):
        host.one_device(3)


def test_float32_rows_of_256_are_split_as_rows_by_themselves(lib) -> None:
    """No tile computes them together, so the splits are those of so many rows, and no list of rows is kept."""
    host = _native.bound_host()
    sizes = lambda rows, dim, dtype, splits=0, n=512: host.window_workspace(n, 8, 2, dim, dtype, 4096, 0, 2512, rows, splits)  # noqa: E731
    assert sizes(512, 256, 0) == sizes(1, 256, 0) == (1, 0)  # 1024 workgroups of one row each fill the CUs
    assert sizes(512, 256, 1)[0] == sizes(512, 128, 0)[0] == lib.pkv_window_splits(512, 8, 2, 4096, 0, 2512, 512) == 16
    assert sizes(512, 256, 0, 3) == (3, 512 * 8 * 3 * 258 * 4)
    assert sizes(5, 256, 0, n=5)[0] == 19  # few of them: 128 keys to a split
    for dim, dtype in ((32, 0), (64, 1), (128, 0), (128, 1), (256, 1)):
        for rows, splits in ((1, 0), (512, 0), (512, 5)):
            got = sizes(rows, dim, dtype, splits)
            assert got[0] == (splits or lib.pkv_window_splits(512, 8, 2, 4096, 0, 2512, rows))
            assert got[1] == lib.pkv_window_workspace_bytes(512, 8, dim, rows, got[0])
    bytes_out = ctypes.c_int64()
    for changes in ({0: -1}, {1: 7}, {2: 0}, {3: 0}, {4: 2}, {5: 0}, {6: -1}, {7: -1}, {8: -1}, {9: -1}, {9: 65}, {10: None}):
        args = [512, 8, 2, 256, 0, 4096, 0, 2512, 512, 0, ctypes.byref(bytes_out)]
        for place, value in changes.items():
            args[place] = value
        assert lib.pkv_window_sizes(*args) == EINVAL, changes


def test_workspace_bytes_serve_every_type(lib) -> None:
    from paged_kv_serving_amd import ops

    host = _native.bound_host()
    for rows, heads, kv_heads in ((512, 8, 2), (30, 45, 1), (700, 45, 1), (1, 8, 8)):
        for dim in (128, 256):
            need = ops.window_workspace_bytes(rows, heads, kv_heads, dim, window=9000, max_context_len=8192)
            each = [host.window_workspace(rows, heads, kv_heads, dim, code, 9000, 0, 8192, rows, 0)[1] for code in (0, 1)]
            assert need == max(each)
    with pytest.raises(ValueError):
        ops.window_workspace_bytes(3, 5, 2, 64, window=9, max_context_len=8)
