"""Block tables that are out of order or out of range in the 8-bit decode attention: reported, nothing else touched."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8
from pagedcore_b200._lib import DEVICE_BAD_BLOCK, check, lib
from tests.fp8_reference import attend64, rope64
from tests.test_fp8_gpu import LAYER, CacheCase, randn

pytestmark = pytest.mark.gpu

GUARD = 1 << 16  # bytes before and behind the workspace


def guarded(size: int, device) -> torch.Tensor:
    return torch.full((GUARD + size + GUARD,), 0x5A, dtype=torch.uint8, device=device)


@pytest.mark.parametrize("prefix", [[0, 3, 2], [-1, 2], [1, 2], [0, -5, 2], [0, 1000000, 2], [0, 90, 40, 60],
                                    [0, 10, 59, 58, 60], [5, 60], [-7, 30, 60], [0, 2**31 - 1, 60]], ids=str)
@pytest.mark.parametrize("layer_call", [False, True])
def test_rows_that_are_out_of_order_are_reported(prefix, layer_call) -> None:
    total, batch = prefix[-1], len(prefix) - 1
    case = CacheCase(151, [16 * 60])
    flat = case.batch()[2][:total].contiguous()
    lengths = torch.full((batch,), 20, dtype=torch.int32, device=case.device)
    table = torch.tensor(prefix, dtype=torch.int32, device=case.device)
    grid, size = fp8.decode_plan(case.device.index, batch, total)
    assert (grid == 1) == (total == 2)
    workspace = guarded(size, case.device)
    out = torch.full((batch + 2, 32, 64), 3.0, dtype=torch.float16, device=case.device)
    query, key, value = (randn(152 + heads, batch, heads, 64).half() for heads in (32, 4, 4))
    new = (key.data_ptr(), value.data_ptr(), 256, case.rope.data_ptr()) if layer_call else ()
    check((lib.pkv_fp8_decode_layer if layer_call else lib.pkv_fp8_decode_attention)(
        *case.cache._args(), LAYER, query.data_ptr(), 2048, *new, lengths.data_ptr(), table.data_ptr(), flat.data_ptr(),
        batch, total, grid, out[1:].data_ptr(), 2048, workspace[GUARD:].data_ptr(), size, case.flag.data_ptr(),
        torch.cuda.current_stream().cuda_stream))
    assert int(case.flag.item()) & DEVICE_BAD_BLOCK
    assert bool((workspace[:GUARD] == 0x5A).all()) and bool((workspace[GUARD + size :] == 0x5A).all())
    assert bool((out[0] == 3).all()) and bool((out[-1] == 3).all())


def test_rows_in_order_are_not_reported() -> None:
    for lengths in ([0, 5, 0, 300, 0], [0], [960], [16] * 60):
        case = CacheCase(153, lengths)
        query = randn(154, len(lengths), 32, 64).half()
        case.check_attention(query, fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag))
        assert int(case.flag.item()) == 0


@pytest.mark.parametrize("lengths, bad", [([40], [(0, 1)]), ([40], [(0, 0), (0, 1), (0, 2)]), ([3, 300, 17], [(1, 0), (1, 7), (2, 1)]),
                                          ([1], [(0, 0)]), ([2048, 64], [(0, 127), (0, 64), (1, 3)]), ([130] * 9, [(4, 8), (8, 2)])],
                         ids=lambda v: "-".join(map(str, v[:3])).replace(" ", ""))
@pytest.mark.parametrize("layer_call", [False, True])
def test_a_bad_block_reads_as_zeros(lengths, bad, layer_call) -> None:
    """A block id outside the cache stands for 16 tokens of zero keys and values, whatever block 0 holds."""
    case = CacheCase(155, lengths)
    case.cache.key_codes.view(torch.uint8)[LAYER, 0] = 0x70  # recognisable: 128, with a scale of 4
    case.cache.value_codes.view(torch.uint8)[LAYER, 0] = 0x70
    case.cache.key_scales[LAYER, 0], case.cache.value_scales[LAYER, 0] = 4.0, 4.0
    for table in case.tables:  # block 0 belongs to nobody
        assert len(case.free) > 1
        if 0 in table:
            at, spare = table.index(0), case.free.pop()
            table[at] = spare
            for name in ("key_codes", "value_codes"):
                getattr(case.cache, name).view(torch.uint8)[LAYER, spare] = 0
            for name in ("key_scales", "value_scales"):
                getattr(case.cache, name)[LAYER, spare] = 1.0
            for oracle in (case.key, case.value):
                oracle.values[spare] = 0.0
    lengths_, prefix, flat, total = case.batch()
    for index, (row, block) in enumerate(bad):
        flat[int(prefix[row]) + block] = (-1, case.cache.num_blocks, 2**31 - 1)[index % 3]
    query = 2 * randn(156, len(lengths), 32, 64).half()
    if layer_call:  # the new token of a row whose last block is bad is not written
        key, value = (randn(157 + i, len(lengths), 4, 64).half() for i in range(2))
        out = fp8.decode_layer(case.cache, LAYER, query, key, value, case.rope, lengths_, prefix, flat, total, case.flag)
        query = rope64(query, case.rope, lengths_.long() - 1)
    else:
        out = fp8.decode_attention(case.cache, LAYER, query, lengths_, prefix, flat, total, case.flag)
    assert int(case.flag.item()) == DEVICE_BAD_BLOCK
    for row, length in enumerate(lengths):
        good = torch.tensor([b if (row, i) not in bad else -1 for i, b in enumerate(case.tables[row])], device=case.device)
        read = fp8.read_blocks(case.cache, LAYER, good.int(), torch.zeros_like(case.flag))  # zeros for bad ids, too
        k, v = (x.reshape(-1, 4, 64)[:length].double() for x in read)
        exact, bound = attend64(query[row], k, v)
        assert bool(((out[row].double() - exact).abs() <= bound).all()), row


@pytest.mark.parametrize("lengths", [[0], [5, 0, 40], [0, 0, 300, 0, 17, 0, 0], [0] * 70 + [2048], [1] + [0] * 300], ids=lambda v: f"{len(v)}rows{max(v)}")
def test_a_decode_layer_row_without_blocks_gives_zeros(lengths) -> None:
    case = CacheCase(158, [max(0, n - 1) for n in lengths])
    for row, length in enumerate(lengths):
        if len(case.tables[row]) * 16 < length:
            case.tables[row].append(case.free.pop())
        case.lengths[row] = length
    rows = len(lengths)
    query, key, value = (randn(159 + heads, rows, heads, 64).half() for heads in (32, 4, 4))
    query[torch.tensor(lengths) == 0] = float("nan")
    calls = []
    for out in (None, torch.full((rows + 1, 40, 64), 7.0, dtype=torch.float16, device=case.device)):
        torch.full((rows, 32, 64), 9.0, dtype=torch.float16, device=case.device)  # storage that the next call may get
        calls.append(fp8.decode_layer(case.cache, LAYER, query, key, value, case.rope, *case.batch(), case.flag,
                                      None if out is None else out[:rows, 4:36]))
    assert int(case.flag.item()) == 0
    assert bool((out[rows] == 7).all()) and bool((out[:, :4] == 7).all()) and bool((out[:, 36:] == 7).all())
    exact_query = rope64(query.nan_to_num(), case.rope, (torch.tensor(lengths, device=case.device) - 1).clamp(min=0))
    for result in calls:
        for row, length in enumerate(lengths):
            blocks = torch.tensor(case.tables[row], dtype=torch.int32, device=case.device)
            k, v = (x.reshape(-1, 4, 64)[:length].double() for x in fp8.read_blocks(case.cache, LAYER, blocks, case.flag))
            exact, bound = attend64(exact_query[row], k, v)
            assert bool(((result[row].double() - exact).abs() <= bound).all()), row


def test_rows_past_a_replayed_batch_are_left_alone() -> None:
    """The entry point that step graphs launch: a row without blocks keeps its output."""
    case = CacheCase(160, [20, 0])
    lengths, prefix, flat, total = case.batch()
    query, key, value = (randn(161 + heads, 2, heads, 64).half() for heads in (32, 4, 4))
    grid, size = fp8.decode_plan(case.device.index, 2, total)
    workspace = torch.empty(size, dtype=torch.uint8, device=case.device)
    for function, kept in ((lib.pkv_fp8_decode_layer, 3.0), (lib.pkv_fp8_decode_layer_zero, 0.0)):
        out = torch.full((2, 32, 64), 3.0, dtype=torch.float16, device=case.device)
        check(function(*case.cache._args(), LAYER, query.data_ptr(), 2048, key.data_ptr(), value.data_ptr(), 256,
                       case.rope.data_ptr(), lengths.data_ptr(), prefix.data_ptr(), flat.data_ptr(), 2, total, grid,
                       out.data_ptr(), 2048, workspace.data_ptr(), size, case.flag.data_ptr(),
                       torch.cuda.current_stream().cuda_stream))
        assert bool((out[1] == kept).all()) and not bool((out[0] == 3.0).any())
