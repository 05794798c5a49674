"""The 4-bit decode operators over more than 1024 rows, whose pieces find their rows in steps."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import int4
from tests.fp8_reference import F32
from tests.int4_reference import LAYER, Case, rope64
from tests.test_int4_gpu import check_rows, randn

pytestmark = pytest.mark.gpu

MIXED = [0, 1, 17, 0, 0, 33, 5, 64, 0, 130, 16, 2]  # lengths, in turn


def lengths_of(rows: int) -> list[int]:
    return [MIXED[(i * 7 + i // 13) % len(MIXED)] for i in range(rows - 1)] + [50]


@pytest.mark.parametrize("rows", [1024, 1025, 1100, 2050])
@pytest.mark.parametrize("layer_call", [False, True])
def test_many_rows_with_empty_ones(rows, layer_call) -> None:
    case = Case(rows, lengths_of(rows))
    query = randn(1, rows, 32, 64).half()
    if not layer_call:
        out = int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
        assert int(case.flag.item()) == 0
        check_rows(case, query.double(), out)
        return
    key, value = randn(2, rows, 4, 64).half(), randn(3, rows, 4, 64).half()
    out = int4.decode_layer(case.cache, LAYER, query, key, value, case.rope, *case.batch(), case.flag)
    positions = torch.tensor(case.lengths, device=case.device) - 1
    k64, q64 = (rope64(x, case.rope, positions.clamp(min=0)) for x in (key, query))
    held = [row for row, length in enumerate(case.lengths) if length]
    slots = torch.cat([case.slots(row, case.lengths[row] - 1, 1) for row in held])
    case.hold(slots, k64[held].float(), value[held].float())
    case.check_values()
    # The rotated query: a rounding to FP32 of each of its steps, and its two halves.
    check_rows(case, q64, out, moved=6 * F32 + 2.0**-22)


def falling(rows: int, total: int, value: int) -> list[int]:
    """A prefix of zeros but for one entry inside the first step and the last one."""
    prefix = [value] * rows + [total]
    prefix[0], prefix[35] = 0, 5
    return prefix


@pytest.mark.parametrize("prefix", [falling(1100, 10, 0), falling(1100, 10, -7), falling(2600, 40, 0), falling(1100, 10, -(2**31))],
                         ids=["zeros", "below zero", "2600 rows", "the lowest"])
@pytest.mark.parametrize("layer_call", [False, True])
def test_many_rows_out_of_order_are_reported_and_read_nothing_before_the_list(prefix, layer_call) -> None:
    rows, total = len(prefix) - 1, prefix[-1]
    case = Case(7, [16 * total], spare=40)
    before = case.cache.storage.clone()
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=case.device)  # noqa: E731
    # Free blocks in front of the list: a row's token written through them would show.
    flat = as_int((case.free * 4)[:16] + case.tables[0])[16:]
    args = (as_int([20] * rows), as_int(prefix), flat, total, case.flag)
    q, k, v = (randn(i, rows, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
    if layer_call:
        int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *args)
    else:
        int4.decode_attention(case.cache, LAYER, q, *args)
    assert int(case.flag.item()) & 1
    untouched = case.free + [case.tables[0][i] for i in range(total) if i + 1 not in prefix]
    assert torch.equal(case.cache.storage[:, untouched], before[:, untouched])
