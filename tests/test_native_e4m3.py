"""What pkv_append_e4m3 and pkv_attention_e4m3 refuse at the C ABI: every refusal returns before any HIP call, so no GPU is
needed and the pointers are made up."""

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
    for kind, star, field in re.findall(r"(?:const )?(\w+)(\*?) (\w+);", body):
        fields.append((field, ctypes.c_void_p if star else getattr(ctypes, {"float": "c_float"}.get(kind, "c_" + kind[:-2]))))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        _native.build()
    return _native.library()


def refused(function, kind, good: dict, **changes) -> int:
    args = kind()
    for name, value in {**good, **changes}.items():
        setattr(args, name, value)
    return function(ctypes.addressof(args), 0, None)


APPEND = dict(
    key_pool=FAKE, value_pool=2 * FAKE, key_scales=3 * FAKE, value_scales=4 * FAKE, keys=5 * FAKE, values=6 * FAKE, key_token_stride=128,
    value_token_stride=128, slot_mapping=7 * FAKE, num_tokens=9, num_blocks=40, src_dtype=0, block_size=16, num_kv_heads=2, head_dim=64,
)  # fmt: skip
ATTENTION = dict(
    out=FAKE, queries=2 * FAKE, query_token_stride=512, query_positions=3 * FAKE, query_seq=4 * FAKE, num_queries=7,
    key_cache=5 * FAKE, value_cache=6 * FAKE, key_scales=10 * FAKE, value_scales=11 * FAKE, num_blocks=40, block_tables=7 * FAKE,
    context_lens=8 * FAKE, workspace=9 * FAKE, workspace_bytes=1 << 20, q_dtype=0, block_size=16, block_table_stride=10, num_seqs=4,
    num_heads=8, num_kv_heads=2, head_dim=64, window=32, sinks=2, max_context_len=160, max_query_len=7, num_splits=2, scale=0.125,
)  # fmt: skip


@pytest.mark.parametrize("changes,code", [
    *(({name: -1}, EINVAL) for name in ("num_tokens", "num_blocks")), *(({name: 0}, EINVAL) for name in ("block_size", "num_kv_heads")),
    *(({name: None}, EINVAL) for name in ("key_pool", "value_pool", "key_scales", "value_scales", "keys", "values", "slot_mapping")),
    *(({name: FAKE + 4}, EINVAL) for name in ("key_pool", "value_pool")), ({"src_dtype": 2}, EINVAL), ({"src_dtype": -1}, EINVAL),
    ({"key_token_stride": 127}, EINVAL), ({"value_token_stride": 0}, EINVAL), ({"head_dim": 48}, EUNSUPPORTED), ({"head_dim": 512}, EUNSUPPORTED),
    ({"num_blocks": 1 << 27}, EUNSUPPORTED), ({"num_blocks": 1 << 62}, EUNSUPPORTED),
    ({"num_tokens": (1 << 31) - 1}, EUNSUPPORTED), ({"num_tokens": (1 << 63) - 1}, EUNSUPPORTED),
    ({"num_kv_heads": 1 << 24, "key_token_stride": 1 << 40, "value_token_stride": 1 << 40}, EUNSUPPORTED),
], ids=str)  # fmt: skip
def test_append_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_append_e4m3, structure("pkv_e4m3_append"), APPEND, **changes) == code


@pytest.mark.parametrize("changes,code", [
    *(({name: -1}, EINVAL) for name in ("num_queries", "num_seqs", "num_blocks", "block_table_stride", "sinks",
                                        "max_context_len", "max_query_len", "num_splits")),
    *(({name: 0}, EINVAL) for name in ("num_heads", "num_kv_heads", "block_size", "window")),
    *(({name: None}, EINVAL) for name in ("out", "queries", "query_positions", "query_seq", "key_cache", "value_cache", "key_scales",
                                          "value_scales", "block_tables", "context_lens", "workspace")),
    *(({name: FAKE + 8}, EINVAL) for name in ("out", "queries", "key_cache", "value_cache", "workspace")),
    ({"num_heads": 7}, EINVAL), ({"num_splits": 65}, EINVAL), ({"max_context_len": 161}, EINVAL), ({"q_dtype": 2}, EINVAL),
    ({"head_dim": 48}, EUNSUPPORTED), ({"num_heads": 130}, EUNSUPPORTED), ({"num_blocks": 1 << 27}, EUNSUPPORTED),
    ({"max_context_len": (1 << 30) + 1, "block_table_stride": 1 << 30}, EUNSUPPORTED),
    ({"query_token_stride": 511}, EINVAL), ({"query_token_stride": 514}, EINVAL), ({"workspace_bytes": 100}, EINVAL),
], ids=str)  # fmt: skip
def test_attention_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_attention_e4m3, structure("pkv_e4m3_attention"), ATTENTION, **changes) == code


def test_the_attentions_workspace(lib) -> None:
    kind = structure("pkv_e4m3_attention")

    def need(**changes) -> int:
        args = kind()
        for name, value in {**ATTENTION, "num_splits": 0, "sinks": 0, **changes}.items():
            setattr(args, name, value)
        return lib.pkv_attention_e4m3_workspace_bytes(ctypes.addressof(args))

    decode = dict(window=(1 << 31) - 1, max_query_len=1, num_queries=64, max_context_len=32768, num_heads=32, num_kv_heads=8, head_dim=128)
    shares = need(**decode)
    assert shares >= 2 * 32 * 130 * 4 * 128 and shares % 16 == 0  # two parts of every head for each of 128 shares
    assert need(**{**decode, "num_queries": 65}) == shares  # whatever the rows
    assert need(**decode, num_splits=1) == 0 and need(**{**decode, "max_context_len": 500}) == 0
    for more in ({"num_splits": 5}, {"block_size": 24}, {"window": 4096}, {"num_blocks": 0}, {"num_queries": 1025}):  # as windowed attention's
        args = {**ATTENTION, "num_splits": 0, "sinks": 0, **decode, **more}
        size = ctypes.c_int64()
        sizes = [args[name] for name in ("num_queries", "num_heads", "num_kv_heads", "head_dim", "q_dtype", "window", "sinks", "max_context_len", "max_query_len",
                                         "num_splits")]  # fmt: skip
        assert lib.pkv_window_sizes(*sizes, ctypes.addressof(size)) >= 1
        assert need(**{**decode, **more}) == size.value
    for bad in ({"num_queries": -1}, {"num_heads": 7}, {"num_kv_heads": 0}, {"block_size": 0}, {"window": 0}, {"num_splits": 65}, {"q_dtype": 2}, {"num_heads": 130}):
        assert need(**bad) == EINVAL
    assert lib.pkv_attention_e4m3_workspace_bytes(None) == EINVAL


@pytest.mark.parametrize("num_queries,max_context_len,shared", [
    (1, 1 << 30, True), (15, 1 << 30, True), (16, 1 << 30, False), (64, (1 << 28) - 16, True), (64, (1 << 28) - 15, False), (64, 1 << 28, False),
    (1024, (1 << 24) - 16, True), (1024, 1 << 24, False), (1024, 1 << 30, False),
])  # fmt: skip
@pytest.mark.parametrize("head_dim", [32, 256])
def test_rows_whose_rounds_32_bits_do_not_count_are_split_by_themselves(lib, num_queries, max_context_len, shared, head_dim) -> None:
    """Equal shares are of the sum of all rows' rounds of 16 keys or more, which has to stay below 2^30."""
    kind, size = structure("pkv_e4m3_attention"), ctypes.c_int64()
    args = kind()
    more = dict(num_queries=num_queries, max_context_len=max_context_len, head_dim=head_dim, num_heads=8, window=(1 << 31) - 1, sinks=0, max_query_len=1, num_splits=0)
    for name, value in {**ATTENTION, **more}.items():
        setattr(args, name, value)
    assert lib.pkv_window_sizes(num_queries, 8, 2, head_dim, 0, (1 << 31) - 1, 0, max_context_len, 1, 0, ctypes.addressof(size)) >= 1
    assert (lib.pkv_attention_e4m3_workspace_bytes(ctypes.addressof(args)) != size.value) == shared


@pytest.mark.parametrize("q_dtype", [0, 1])
@pytest.mark.parametrize("num_splits", [0, 1, 2])
def test_the_workspace_of_a_call_without_queries(lib, q_dtype, num_splits) -> None:
    """A plan without rows, whatever their runs would be: what windowed attention needs, and no division by no tiles."""
    from paged_kv_serving_amd import ops

    kind, size = structure("pkv_e4m3_attention"), ctypes.c_int64()
    for max_query_len in (0, 1, 4, 512, (1 << 31) - 1):
        for heads, window, num_seqs in ((8, 100, 0), (64, (1 << 31) - 1, 4), (128, 8, 1)):
            args = kind()
            more = dict(num_queries=0, q_dtype=q_dtype, num_splits=num_splits, max_query_len=max_query_len, num_heads=heads, window=window, sinks=0, num_seqs=num_seqs)
            for name, value in {**ATTENTION, **more}.items():
                setattr(args, name, value)
            sizes = (0, heads, 2, 64, q_dtype, window, 0, 160, max_query_len, num_splits)
            assert lib.pkv_window_sizes(*sizes, ctypes.addressof(size)) >= 1
            assert lib.pkv_attention_e4m3_workspace_bytes(ctypes.addressof(args)) == size.value
        assert ops.e4m3_workspace_bytes(0, 8, 2, 64, block_size=16, max_context_len=160, max_query_len=max_query_len, num_splits=num_splits) == size.value


def test_no_arguments_and_nothing_to_do(lib) -> None:
    for function in (lib.pkv_append_e4m3, lib.pkv_attention_e4m3):
        assert function(None, 0, None) == EINVAL
    assert refused(lib.pkv_append_e4m3, structure("pkv_e4m3_append"), APPEND, num_tokens=0) == 0
    assert refused(lib.pkv_attention_e4m3, structure("pkv_e4m3_attention"), ATTENTION, num_queries=0) == 0


def test_tensors_off_the_device_are_refused_by_name(lib) -> None:
    import torch

    from paged_kv_serving_amd import ops

    f, i32, i64 = torch.zeros(1, 2, 32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    pool, table, scales = torch.zeros(4, 8, 2, 32, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(4, 2)
    with pytest.raises(ValueError, match="HIP device"):
        ops.append_kv_e4m3(pool, pool, scales, scales, f, f, i64)
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_attention_e4m3(f, i32, i32, pool, pool, scales, scales, table, i32, 1.0, max_context_len=8)
