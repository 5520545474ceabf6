"""What pkv_step_metadata, pkv_beam_select and pkv_beam_reorder refuse at the C ABI, and the selection's host function: every
refusal returns before any HIP call, so no GPU is needed and the pointers are made up."""

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
        fields.append((field, c_type * int(re.search(rf"#define {count} (\d+)", HEADER).group(1)) if count else c_type))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        _native.build()
    return _native.library()


def refused(function, kind, good: dict, **changes) -> int:
    args = kind()
    for name, value in {**good, **changes}.items():
        if isinstance(value, (list, tuple)):
            for i, one in enumerate(value):
                getattr(args, name)[i] = one
        else:
            setattr(args, name, value)
    return function(ctypes.addressof(args), 0, None)


STEP = dict(
    query_lens=FAKE, context_lens=2 * FAKE, block_tables=3 * FAKE, free_blocks=4 * FAKE, next_free=5 * FAKE, query_seq=6 * FAKE,
    query_positions=7 * FAKE, positions=8 * FAKE, slot_mapping=9 * FAKE, query_starts=10 * FAKE, context_lens_out=11 * FAKE,
    next_free_out=12 * FAKE, num_rows=30, num_seqs=4, table_stride=10, num_free=20, block_size=16,
)  # fmt: skip
BEAM = dict(
    best_scores=FAKE, best_beams=2 * FAKE, best_tokens=3 * FAKE, logits=4 * FAKE, row_stride=100, num_groups=3, vocab_size=100,
    scores=5 * FAKE, workspace=6 * FAKE, workspace_bytes=1 << 20, dtype=0, num_beams=4, count=8,
)  # fmt: skip
REORDER = dict(
    new_tables=FAKE, block_tables=2 * FAKE, parents=3 * FAKE, context_lens=4 * FAKE, num_groups=3, num_blocks=40, states=[5 * FAKE],
    block_bytes=[64], layer_bytes=[2560], num_layers=[2], num_states=1, num_beams=4, table_stride=10, block_size=16,
)  # fmt: skip


@pytest.mark.parametrize("changes,code", [
    *(({name: -1}, EINVAL) for name in ("num_rows", "num_seqs", "table_stride", "num_free")), ({"block_size": 0}, EINVAL),
    *(({name: None}, EINVAL) for name in STEP if name not in ("next_free", "num_rows", "num_seqs", "table_stride", "num_free", "block_size")),
    ({"num_rows": (1 << 21) + 1}, EUNSUPPORTED), ({"num_rows": 1 << 62}, EUNSUPPORTED), ({"num_free": (1 << 29) + 1}, EUNSUPPORTED),
    ({"table_stride": 1 << 20, "block_size": 1 << 12}, EUNSUPPORTED), ({"next_free_out": 5 * FAKE}, EINVAL), ({"context_lens_out": 2 * FAKE}, EINVAL),
], ids=str)  # fmt: skip
def test_step_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_step_metadata, structure("pkv_step"), STEP, **changes) == code


@pytest.mark.parametrize("output,size", [
    ("query_seq", 120), ("query_positions", 120), ("positions", 240), ("slot_mapping", 240), ("query_starts", 20), ("context_lens_out", 16),
    ("next_free_out", 4), ("block_tables", 160),
])  # fmt: skip
@pytest.mark.parametrize("read,bytes_read", [("query_lens", 16), ("context_lens", 16), ("free_blocks", 80), ("next_free", 4)])
def test_step_outputs_in_the_memory_of_an_input_are_refused(lib, output, size, read, bytes_read) -> None:
    for away in (4 - size, 0, bytes_read - 4):
        assert refused(lib.pkv_step_metadata, structure("pkv_step"), STEP, **{output: STEP[read] + away}) == EINVAL


@pytest.mark.parametrize("changes,code", [
    ({"num_groups": -1}, EINVAL), ({"num_beams": 0}, EINVAL), ({"vocab_size": 0}, EINVAL), ({"count": 0}, EINVAL), ({"dtype": 2}, EINVAL),
    ({"row_stride": 99}, EINVAL), ({"num_beams": 65}, EUNSUPPORTED), ({"count": 129}, EUNSUPPORTED), ({"num_groups": 1 << 19}, EUNSUPPORTED),
    ({"num_groups": 1 << 62}, EUNSUPPORTED), ({"vocab_size": 1 << 26, "row_stride": 1 << 26}, EUNSUPPORTED), ({"vocab_size": 1, "count": 5}, EINVAL),
    ({"workspace_bytes": 100}, EINVAL), ({"workspace": 6 * FAKE + 8}, EINVAL),
    *(({name: None}, EINVAL) for name in ("best_scores", "best_beams", "best_tokens", "logits", "scores", "workspace")),
], ids=str)  # fmt: skip
def test_select_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_beam_select, structure("pkv_beam"), BEAM, **changes) == code


@pytest.mark.parametrize("changes,code", [
    *(({name: -1}, EINVAL) for name in ("num_groups", "num_blocks", "table_stride", "num_states")), ({"num_beams": 0}, EINVAL), ({"block_size": 0}, EINVAL),
    *(({name: [-1]}, EINVAL) for name in ("num_layers", "block_bytes", "layer_bytes")), ({"states": [None]}, EINVAL), ({"num_beams": 65}, EUNSUPPORTED),
    ({"num_states": 9}, EUNSUPPORTED), ({"num_layers": [65536]}, EUNSUPPORTED), ({"num_groups": 1 << 40}, EUNSUPPORTED),
    ({"table_stride": 1 << 20, "block_size": 1 << 12}, EUNSUPPORTED), ({"new_tables": 2 * FAKE}, EINVAL),
    *(({name: None}, EINVAL) for name in ("new_tables", "block_tables", "parents", "context_lens")),
], ids=str)  # fmt: skip
def test_reorder_refusals(lib, changes, code) -> None:
    assert refused(lib.pkv_beam_reorder, structure("pkv_reorder"), REORDER, **changes) == code


@pytest.mark.parametrize("away", [-476, -4, 0, 4, 40, 476])
def test_tables_that_share_memory_are_refused(lib, away) -> None:
    """3 groups of 4 rows of 10 entries, 480 bytes: no entry of the output may be one of the input."""
    assert refused(lib.pkv_beam_reorder, structure("pkv_reorder"), REORDER, new_tables=2 * FAKE + away) == EINVAL


@pytest.mark.parametrize("count,away", [(8, -23 * 4), (8, -4), (8, 0), (8, 4), (8, 11 * 4), (4, -11 * 4), (4, 4), (4, 11 * 4), (2, 0)])
def test_best_scores_in_the_memory_of_the_scores_are_refused(lib, count, away) -> None:
    """3 groups of 4 beams: 12 scores, 3 * count best ones."""
    assert refused(lib.pkv_beam_select, structure("pkv_beam"), BEAM, count=count, best_scores=5 * FAKE + away) == EINVAL


def test_no_arguments_and_nothing_to_do(lib) -> None:
    for function in (lib.pkv_step_metadata, lib.pkv_beam_select, lib.pkv_beam_reorder):
        assert function(None, 0, None) == EINVAL
    assert refused(lib.pkv_beam_select, structure("pkv_beam"), BEAM, num_groups=0) == 0
    assert refused(lib.pkv_beam_reorder, structure("pkv_reorder"), REORDER, num_groups=0) == 0


def test_the_selections_workspace(lib) -> None:
    size = lib.pkv_beam_workspace_bytes
    for groups, beams, vocab, count in ((1, 1, 1, 1), (1, 4, 32000, 8), (32, 8, 128256, 16), (3, 64, 50257, 128)):
        per_chunk = 8 + 4 + 8 * count
        # A chunk is 2,048 logits where rows are few, else 8,192.
        most, least = (-(-vocab // n) * groups * beams * per_chunk for n in (2048, 8192))
        assert least <= size(groups, beams, vocab, count) <= most + 15 and size(groups, beams, vocab, count) % 16 == 0
    assert size(0, 4, 100, 8) == 0
    for bad in ((-1, 1, 1, 1), (1, 0, 1, 1), (1, 65, 1, 1), (1, 1, 0, 1), (1, 1, 1 << 26, 1), (1, 1, 1, 0), (1, 1, 1, 129), (1 << 20, 2, 9, 1),
                (1, 64, 1 << 20, 1)):  # fmt: skip
        assert size(*bad) == EINVAL


def test_tensors_off_the_device_are_refused_by_name(lib) -> None:
    import torch

    from paged_kv_serving_amd import ops

    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="HIP device"):
        ops.step_metadata(i32(2), i32(2), i32(2, 4), i32(3), block_size=16, num_rows=4)
    with pytest.raises(ValueError, match="HIP device"):
        ops.beam_select(torch.zeros(4, 9), torch.zeros(4), num_beams=2)
    with pytest.raises(ValueError, match="HIP device"):
        ops.beam_reorder(i32(4, 3), i32(2, 2), i32(2), [], block_size=4)
