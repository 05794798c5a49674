"""The 4-bit KV cache: write, read back and attention against 64-bit arithmetic."""

from __future__ import annotations

import math

import pytest
import torch

from pagedcore_b200 import int4
from tests.conftest import cuda_device
from tests.fp8_reference import F32, HALF_FP16, attend64
from tests.int4_reference import LAYER, LAYERS, Case, norm64, rope64, scale_for, stored, unpack

pytestmark = pytest.mark.gpu

# The kernels' norm of a query head in FP32: 16 squares a lane and two sums over lanes (18
# roundings, halved by the root), the root (2 ulp) and two products; a rotation adds three.
NORM_ERROR = 16 * F32


def randn(seed: int, *shape: int) -> torch.Tensor:
    device = cuda_device()
    return torch.randn(shape, device=device, generator=torch.Generator(device=device).manual_seed(seed))


def head_norms(seed: int) -> int4.HeadNorms:
    return int4.HeadNorms(*((1 + 0.2 * randn(seed + i, LAYERS, 64)).half() for i in range(2)), 1e-5)


def check_rows(case: Case, query64: torch.Tensor, out: torch.Tensor, moved: float = 0.0) -> None:
    """``out`` is the attention of query64 [rows, 32, 64], itself off by ``moved`` of its rows' largest values."""
    for row, length in enumerate(case.lengths):
        key, value = case.tokens(row)
        exact, bound = attend64(query64[row], key, value)
        if moved and length:
            size = query64[row].abs().amax(-1).view(4, 8, 1)
            off = moved * size * key.abs().sum(-1).amax(0)[:, None, None] / 8  # of any score
            bound = bound + (2 * off * value.abs().amax(0)[:, None]).reshape(32, 64)
        assert bool(((out[row].double() - exact).abs() <= bound).all()), (row, length)


# -- write and read ------------------------------------------------------------------
def test_append_and_read() -> None:
    case = Case(1, [40, 1, 16, 33])
    case.check_values()
    for row in range(4):
        if case.lengths[row] % 16 == 0:
            case.tables[row].append(case.free.pop())
        case.append(row, 50 * randn(90 + row, 1, 4, 64), 300 * randn(95 + row, 1, 4, 64), case.lengths[row])
        case.lengths[row] += 1
    case.check_values()
    case.tables[0] += [case.free.pop(), case.free.pop()]
    case.append(0, randn(77, 37, 4, 64), randn(78, 37, 4, 64), 41)  # from inside a block
    case.lengths[0] += 37
    case.check_values()


@pytest.mark.parametrize("factor", [2.0**-24, 2.0**-20, 2.0**-17, 2.0**-13, 2.0**-11, 1.0, 1000.0, 15000.0])
def test_append_over_the_whole_range_of_fp16(factor) -> None:
    """Every value ends within half a step; steps are 2^-17 or more, and past 64512 values stay there."""
    case = Case(2, [64])
    key, value = (torch.clamp(randn(i, 64, 4, 64) * factor, -65504, 65504).half().float() for i in (3, 4))
    case.append(0, key, value, 0)
    case.check_values()
    for got, rows in zip(case.tokens(0), (key, value)):
        step = scale_for(rows.unflatten(-1, (4, 16)).abs().amax(-1)).repeat_interleave(16, -1)
        assert bool(((got - rows.clamp(-64512, 64512).double()).abs() <= step / 2).all())


def test_append_at_ties_and_ends() -> None:
    """Values in the middle between two codes, scales between two numbers, zeros, one value alone in a group."""
    case = Case(3, [48])
    grid = torch.arange(-56, 57, device=case.device) / 8.0  # multiples of an eighth: halves fall on ties
    key = grid[torch.randint(0, 113, (48, 4, 64), device=case.device, generator=torch.Generator(case.device).manual_seed(1))]
    key[..., ::16] = 7.0
    value = torch.zeros(48, 4, 64, device=case.device)
    scales = torch.linspace(8, 16, 48, device=case.device)[:, None] * torch.exp2(torch.arange(4, device=case.device))[None]
    value[..., 5::16] = 7 * scales[..., None] / 8  # sevenths between and on the numbers
    value[7] = 0
    value[8, :, ::16] = 65504
    case.append(0, key, value, 0)
    case.check_values()


def test_the_bytes_are_the_documented_ones() -> None:
    case = Case(4, [20])
    key, value = case.tokens(0)
    for token, head in ((0, 0), (5, 3), (15, 2), (19, 1)):
        parts = unpack(case.cache.storage[LAYER], case.tables[0][token // 16], head, token % 16)
        for codes, scales, want in ((*parts[:2], key[token, head]), (*parts[2:], value[token, head])):
            got = [c * math.ldexp(s % 8 + 8 * (s > 7), max(s // 8, 1) - 18) for c, s in
                   zip(codes, [s for s in scales for _ in range(16)])]
            assert got == want.tolist()


def test_append_leaves_everything_else_as_it_was() -> None:
    case = Case(5, [20, 5])
    before = case.cache.storage.clone()
    case.append(0, 9 * randn(3, 3, 4, 64), 9 * randn(4, 3, 4, 64), 20)
    case.lengths[0] = 23
    case.check_values()
    changed = (case.cache.storage != before).view(LAYERS, -1, 4, 1152)
    block = case.tables[0][1]
    assert not bool(changed[[0, 2]].any())
    others = [b for b in range(case.cache.num_blocks) if b != block]
    assert not bool(changed[LAYER, others].any())
    heads = changed[LAYER, block]
    for at, parts, width in ((0, 4, 8), (512, 8, 4), (1024, 4, 1), (1088, 4, 1)):
        tokens = heads[:, at : at + parts * 16 * width].view(4, parts, 16, width)
        assert not bool(tokens[:, :, [*range(4), *range(7, 16)]].any())


def test_append_takes_any_order_several_layers_and_strides() -> None:
    case = Case(6, [0], spare=8)
    case.tables[0] = case.free[:5]
    order = torch.randperm(80, generator=torch.Generator().manual_seed(1))[:33]
    slots = case.slots(0, 0, 80)[order.to(case.device)]
    wide = randn(7, 33, LAYERS, 12, 64).half()  # token-major, several heads: strides that are not the usual ones
    key, value = wide[:, :, 1:5].transpose(0, 1), wide[:, :, 6:10].transpose(0, 1)
    int4.append_kv(case.cache, key, value, slots, layer_begin=0, error_flag=case.flag)
    blocks = torch.tensor(case.tables[0], dtype=torch.int32, device=case.device)
    for layer in range(LAYERS):
        for got, rows in zip(int4.read_blocks(case.cache, layer, blocks, case.flag), (key, value)):
            got = got.reshape(-1, 4, 64)[order.to(case.device)]
            assert torch.equal(got.double(), stored(rows[layer].float()))
    assert int(case.flag.item()) == 0
    int4.append_kv(case.cache, key[:, :0], value[:, :0], slots, layer_begin=0, error_flag=case.flag)  # no tokens
    assert int4.read_blocks(case.cache, 0, blocks[:0], case.flag)[0].shape == (0, 16, 4, 64)


def test_a_group_that_is_not_finite_reads_as_nan() -> None:
    case = Case(7, [3])
    key, value = randn(5, 2, 4, 64), randn(6, 2, 4, 64)
    key[0, 1, 7], value[1, 2, 9], value[0, 2, 25] = math.inf, math.nan, -math.inf
    case.append(0, key, value, 3)
    case.tables[0] = case.tables[0][:1]
    case.lengths[0] = 5
    case.check_values()
    got = case.tokens(0)
    assert int(got[0].isnan().sum()) == 16 and int(got[1].isnan().sum()) == 32


@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 100), (5, 3), (16, 16), (31, 50), (2040, 8)])
@pytest.mark.parametrize("out", ["fp32", "half", "in place"])
@pytest.mark.parametrize("normed", [False, True])
def test_append_norms_and_rotates(start, tokens, out, normed) -> None:
    case = Case(8, [0], spare=-(-(start + tokens) // 16) + 1)
    case.tables[0] = case.free[: -(-(start + tokens) // 16)]
    wide = randn(9, LAYERS - 1, tokens, 40, 64).half()  # a fused projection's rows
    query, key, value = wide[:, :, :32], wide[:, :, 32:36], wide[:, :, 36:]
    source = query.double()
    positions = torch.arange(start, start + tokens, device=case.device)
    norms = head_norms(11) if normed else None
    query_out = {"fp32": None, "half": torch.empty(LAYERS - 1, tokens, 32, 64, dtype=torch.float16, device=case.device),
                 "in place": query}[out]
    rotated = int4.append_kv(
        case.cache, key, value, case.slots(0, start, tokens), layer_begin=1, error_flag=case.flag,
        positions=positions.int(), rope_table=case.rope, query=query, query_out=query_out, norms=norms,
    )
    assert rotated.dtype is (torch.float32 if out == "fp32" else torch.float16)
    blocks = torch.tensor(case.tables[0], dtype=torch.int32, device=case.device)
    for index in range(LAYERS - 1):
        layer = 1 + index
        q, k = source[index], key[index].double()
        error = 3 * F32
        if normed:
            q, k = norm64(q, norms.query[layer], norms.eps), norm64(k, norms.key[layer], norms.eps)
            error += NORM_ERROR
        exact = rope64(q, case.rope, positions)
        size = q.abs() + q.abs().roll(32, -1)
        bound = error * size + (0 if out == "fp32" else HALF_FP16 * exact.abs() + 2.0**-25)
        assert bool(((rotated[index].double() - exact).abs() <= bound).all())
        got_k, got_v = (x.reshape(-1, 4, 64)[start : start + tokens].double()
                        for x in int4.read_blocks(case.cache, layer, blocks, case.flag))
        assert torch.equal(got_v, stored(value[index].float()))
        k64 = rope64(k, case.rope, positions)
        if normed:
            # FP64, rounded to FP32: the scale is that of an amax off by 2^-23, a value within half of it.
            groups = k64.unflatten(-1, (4, 16)).abs().amax(-1)
            step = torch.maximum(scale_for(groups * (1 - 2.0**-23)), scale_for(groups * (1 + 2.0**-23)))
            assert bool(((got_k - k64).abs() <= step.repeat_interleave(16, -1) * (0.5 + 2.0**-20)).all())
            assert float((got_k == stored(k64.float())).double().mean()) > 0.999
        else:
            assert torch.equal(got_k, stored(k64.float()))
    assert int(case.flag.item()) == 0


def test_appends_outside_the_cache_and_the_rotation_table_are_reported() -> None:
    case = Case(10, [20])
    before = case.cache.storage.clone()
    key, value = randn(1, 1, 3, 4, 64).half(), randn(2, 1, 3, 4, 64).half()
    as_int = lambda *x: torch.tensor(x, dtype=torch.int32, device=case.device)  # noqa: E731
    slots = as_int(-1, 16 * case.cache.num_blocks, 2**31 - 1)
    int4.append_kv(case.cache, key, value, slots, layer_begin=LAYER, error_flag=case.flag)
    assert int(case.flag.item()) == 1 and torch.equal(case.cache.storage, before)
    case.flag.zero_()
    int4.append_kv(case.cache, key, value, case.slots(0, 0, 3), layer_begin=LAYER, error_flag=case.flag,
                   positions=as_int(-1, 2048, 5), rope_table=case.rope)
    assert int(case.flag.item()) == 2
    case.flag.zero_()
    blocks = as_int(case.tables[0][0], -1, case.cache.num_blocks)
    key, value = int4.read_blocks(case.cache, LAYER, blocks, case.flag)
    assert int(case.flag.item()) == 1 and not bool(key[1:].any()) and not bool(value[1:].any())


# -- one token a row -------------------------------------------------------------------
LENGTHS = [[1], [15], [16], [17], [64], [65], [0], [0, 0, 5, 0], [3, 0, 200, 64, 1, 0], [2048], [100, 513, 2048, 17],
           [1] * 70, [33, 64, 1, 128, 127, 129] * 11, [0] * 40 + [700], [9000, 3], [40000],
           [5, 0] * 49, [16 * n + 1 for n in range(8)] * 12, [129] + [3] * 60, [128] * 256, [20] * 300, [128], [129]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}rows{max(v)}")
def test_decode_attention(lengths) -> None:
    case = Case(sum(lengths) + len(lengths), lengths)
    query = randn(9, len(lengths), 32, 64).half()
    out = int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    assert int(case.flag.item()) == 0
    check_rows(case, query.double(), out)
    assert torch.equal(int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag), out)


@pytest.mark.parametrize("rows", [[300, 5, 64], [5, 100, 128], [65, 0, 0], [40, 200, 3]], ids=str)
def test_decode_attention_does_not_depend_on_the_room_of_the_block_list(rows) -> None:
    case = Case(16, rows)
    lengths, prefix, flat, total = case.batch()
    query = randn(3, 3, 32, 64).half()
    expected = int4.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total, case.flag)
    room = torch.cat((flat, torch.full((5000,), -7, dtype=torch.int32, device=case.device)))
    out = int4.decode_attention(case.cache, LAYER, query, lengths, prefix, room, room.numel(), case.flag)
    assert int(case.flag.item()) == 0
    assert torch.equal(out, expected)
    int4.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total - 1, case.flag)  # too little room
    assert int(case.flag.item()) == 1


def test_decode_attention_with_tokens_of_very_different_size() -> None:
    case = Case(12, [300, 90], spread=4.0)
    query = 2 * randn(10, 2, 32, 64).half()
    check_rows(case, query.double(), int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag))


@pytest.mark.parametrize("factor", [2.0**-24, 2.0**-10, 2.0**8, 2.0**14])
@pytest.mark.parametrize("layer_call", [False, True])
def test_decode_attention_of_queries_and_keys_far_out(factor, layer_call) -> None:
    """Queries and K times ``factor`` each: scores from nothing to 2^28 and more."""
    case = Case(17, [100, 333])
    for row, length in enumerate(case.lengths):
        case.append(row, (randn(row, length, 4, 64) * factor).clamp(-65504, 65504), randn(row + 5, length, 4, 64), 0)
    query = (randn(3, 2, 32, 64) * factor).clamp(-65504, 65504).half()
    if not layer_call:
        check_rows(case, query.double(), int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag))
        return
    key, value = (randn(8, 2, 4, 64) * factor).clamp(-65504, 65504).half(), randn(9, 2, 4, 64).half()
    out = int4.decode_layer(case.cache, LAYER, query, key, value, case.rope, *case.batch(), case.flag)
    positions = torch.tensor(case.lengths, device=case.device) - 1
    for row in range(2):
        case.hold(case.slots(row, case.lengths[row] - 1, 1), rope64(key[row : row + 1], case.rope, positions[row : row + 1]).float(),
                  value[row : row + 1].float())
    case.check_values()
    # The rotated query: a rounding to FP32 and the two halves' 2^-22; the softmax is steep, its largest
    # weight may pass from one token to another within this.
    check_rows(case, rope64(query, case.rope, positions), out, moved=2.0**-21)


def test_decode_attention_strides_and_rows_behind_the_last() -> None:
    case = Case(13, [70, 20, 5])
    wide = randn(11, 3, 48, 64).half()
    query = wide[:, 8:40]
    out = torch.full((5, 40, 64), 3.0, dtype=torch.float16, device=case.device)
    result = int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag, out[:3, :32])
    check_rows(case, query.double(), result)
    assert bool((out[3:] == 3).all()) and bool((out[:, 32:] == 3).all())
    expected = result.clone()
    unaligned = torch.empty(3 * 2048 + 1, dtype=torch.float16, device=case.device)[1:].view(3, 32, 64).copy_(query)
    assert torch.equal(int4.decode_attention(case.cache, LAYER, unaligned, *case.batch(), case.flag), expected)
    one = query[:1].expand(3, 32, 64)  # the same row three times
    assert torch.equal(int4.decode_attention(case.cache, LAYER, one, *case.batch(), case.flag),
                       int4.decode_attention(case.cache, LAYER, one.contiguous(), *case.batch(), case.flag))


def test_decode_attention_is_nan_only_where_the_cache_is() -> None:
    case = Case(14, [40, 40, 40])
    key, value = randn(1, 1, 4, 64), randn(2, 1, 4, 64)
    key[0, 2, 5], value[0, 0, 20] = math.nan, math.inf
    case.append(0, key, randn(2, 1, 4, 64), 40)
    case.append(1, randn(1, 1, 4, 64), value, 40)
    case.lengths[:2] = [41, 41]
    out = int4.decode_attention(case.cache, LAYER, randn(15, 3, 32, 64).half(), *case.batch(), case.flag).isnan()
    assert bool(out[0, 16:24].all()) and int(out[0].sum()) == 8 * 64
    assert bool(out[1, :8, 16:32].all()) and int(out[1].sum()) == 8 * 16
    assert not bool(out[2].any())


def test_a_block_outside_the_cache_reads_as_zeros() -> None:
    case = Case(15, [40, 700])
    lengths, prefix, flat, total = case.batch()
    query = randn(1, 2, 32, 64).half()
    flat[1], flat[30] = case.cache.num_blocks, -5
    out = int4.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total, case.flag)
    assert int(case.flag.item()) == 1
    for row, (start, end) in ((0, (16, 32)), (1, (27 * 16, 28 * 16))):
        key, value = (x.clone() for x in case.tokens(row))
        key[start:end] = value[start:end] = 0
        exact, bound = attend64(query[row], key, value)
        assert bool(((out[row].double() - exact).abs() <= bound).all())


@pytest.mark.parametrize(
    "prefix", [[0, 3, 2], [-1, 2], [1, 2], [0, -5, 2], [-5, -2, 2], [-9, -1, 0, 2], [0, 1000000, 2], [0, 90, 40, 60]], ids=str
)
@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("layer_call", [False, True])
def test_rows_out_of_order_are_reported(prefix, layer_call, exact) -> None:
    case = Case(18, [16 * 60])
    count = len(prefix) - 1
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=case.device)  # noqa: E731
    flat = case.batch()[2]
    args = (as_int([20] * count), as_int(prefix), flat, prefix[-1] if exact else flat.numel(), case.flag)
    q, k, v = (randn(i, count, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
    if layer_call:
        int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *args)
    else:
        int4.decode_attention(case.cache, LAYER, q, *args)
    assert int(case.flag.item()) & 1


@pytest.mark.parametrize("lengths", [[1], [16, 17], [1, 15, 16, 48, 700, 65], [2048, 3], [33] * 300, [5] * 49, [130] + [3] * 60], ids=lambda v: f"{len(v)}rows{max(v)}")
@pytest.mark.parametrize("normed", [False, True])
def test_decode_layer_writes_as_append_does_and_attends(lengths, normed) -> None:
    whole, parts = (Case(21, [n - 1 for n in lengths], spare=len(lengths) + 3) for _ in range(2))
    for case in (whole, parts):
        for row, length in enumerate(lengths):
            if len(case.tables[row]) * 16 < length:
                case.tables[row].append(case.free.pop())
            case.lengths[row] = length
    count = len(lengths)
    fused = randn(22, count, 40, 64).half()
    query, key, value = fused[:, :32], fused[:, 32:36], fused[:, 36:]
    norms = head_norms(23) if normed else None
    out = int4.decode_layer(whole.cache, LAYER, query, key, value, whole.rope, *whole.batch(), whole.flag, norms=norms)
    slots = torch.cat([parts.slots(row, n - 1, 1) for row, n in enumerate(lengths)])
    positions = torch.tensor(lengths, dtype=torch.int32, device=parts.device) - 1
    int4.append_kv(parts.cache, key[None], value[None], slots, layer_begin=LAYER, error_flag=parts.flag,
                   positions=positions, rope_table=parts.rope, norms=norms)
    assert torch.equal(whole.cache.storage, parts.cache.storage)
    assert int(whole.flag.item()) == 0
    for row, length in enumerate(lengths):  # what the cache holds now, as read back
        blocks = torch.tensor(whole.tables[row], dtype=torch.int32, device=whole.device)
        for name, got in zip(("key", "value"), int4.read_blocks(whole.cache, LAYER, blocks, whole.flag)):
            whole.held[name][whole.tables[row]] = got.double()
    q64 = norm64(query, norms.query[LAYER], norms.eps) if normed else query.double()
    # Norm and rotation of the query, and its two halves.
    check_rows(whole, rope64(q64, whole.rope, positions.long()), out, moved=(NORM_ERROR if normed else 0) + 6 * F32 + 2.0**-22)


@pytest.mark.parametrize("lengths", [[0], [5, 0, 40], [0, 0, 300, 0, 17, 0, 0], [0] * 70 + [2048], [1] + [0] * 300], ids=lambda v: f"{len(v)}rows{max(v)}")
def test_a_decode_layer_row_without_blocks_gives_zeros(lengths) -> None:
    case = Case(24, lengths)
    q, k, v = (randn(i, len(lengths), h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
    out = torch.full((len(lengths), 32, 64), math.nan, dtype=torch.float16, device=case.device)
    int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *case.batch(), case.flag, out)
    for row, length in enumerate(lengths):
        assert bool((out[row] == 0).all()) if not length else bool(out[row].isfinite().all())
    assert int(case.flag.item()) == 0


def test_decode_layer_reports_a_row_without_a_token() -> None:
    case = Case(25, [0, 20])
    case.tables[0].append(case.free.pop())
    before = case.cache.storage[LAYER, case.tables[0][0]].clone()
    q, k, v = (randn(i, 2, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
    out = int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *case.batch(), case.flag)
    assert int(case.flag.item()) & 2
    assert torch.equal(case.cache.storage[LAYER, case.tables[0][0]], before)
    assert not bool(out[0].any())  # its block has no valid token


# -- a prompt chunk ----------------------------------------------------------------------
@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 15), (0, 130), (7, 40), (64, 3), (100, 64), (601, 75), (300, 500), (2000, 48), (2047, 1), (0, 2047), (0, 75), (20, 90), (700, 330), (1500, 220), (1024, 512), (1039, 701)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prefill_attention(start, tokens, dtype) -> None:
    case = Case(31, [start + tokens])
    query = randn(32, tokens, 32, 64).to(dtype)
    blocks = case.batch()[2]
    wide = torch.full((tokens + 1, 40, 64), 3.0, dtype=torch.float16, device=case.device)
    out = int4.prefill_attention(case.cache, LAYER, query, blocks, start, case.flag, wide[:tokens, 4:36])
    assert int(case.flag.item()) == 0
    for t in {0, 1, tokens // 2, tokens - 1} & set(range(tokens)):
        exact, bound = attend64(query[t], *case.tokens(0, start + t + 1), HALF_FP16)
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t
    assert bool((wide[tokens] == 3).all()) and bool((wide[:, :4] == 3).all()) and bool((wide[:, 36:] == 3).all())
    assert torch.equal(int4.prefill_attention(case.cache, LAYER, query, blocks, start, case.flag), out)


def test_a_prompt_a_bad_block_and_its_report() -> None:
    case = Case(33, [100])
    blocks = case.batch()[2].clone()
    query = randn(34, 100, 32, 64)
    blocks[3] = -1
    out = int4.prefill_attention(case.cache, LAYER, query, blocks, 0, case.flag)
    assert int(case.flag.item()) == 1
    key, value = (x.clone() for x in case.tokens(0))
    key[48:64] = value[48:64] = 0
    exact, bound = attend64(query[99], key, value, HALF_FP16)
    assert bool(((out[99].double() - exact).abs() <= bound).all())


@pytest.mark.parametrize("start, tokens", [(64, 40), (700, 9)])
def test_a_few_prompt_tokens_behind_a_long_context_and_a_bad_block(start, tokens) -> None:
    case = Case(35, [start + tokens])
    blocks, query = case.batch()[2].clone(), randn(36, tokens, 32, 64)
    blocks[2] = case.cache.num_blocks + 5
    out = int4.prefill_attention(case.cache, LAYER, query, blocks, start, case.flag)
    assert int(case.flag.item()) == 1
    for t in (0, tokens - 1):
        key, value = (x.clone() for x in case.tokens(0, start + t + 1))
        key[32:48] = value[32:48] = 0
        exact, bound = attend64(query[t], key, value)
        assert bool(((out[t].double() - exact).abs() <= bound).all())


@pytest.mark.parametrize("exponent", [-60, 16, 24, 31, 60, 100])
@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 40), (0, 200), (300, 70), (1000, 3), (1100, 300)])
def test_prompt_queries_of_any_size(exponent, start, tokens) -> None:
    """Far out the largest score's value alone is left; scores within their rounding of it may take its place."""
    case = Case(37, [start + tokens])
    query = torch.ldexp(randn(38, tokens, 32, 64), torch.tensor(exponent, device=case.device))
    out = int4.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert bool(out.isfinite().all()) and int(case.flag.item()) == 0
    for t in (0, tokens - 1):
        key, value = case.tokens(0, start + t + 1)
        exact, bound = attend64(query[t], key, value, HALF_FP16)
        scores = (query[t].double().view(4, 8, 64) @ key.transpose(0, 1).transpose(1, 2) / 8).topk(min(2, key.shape[0]), -1)[0]
        gap = scores[..., 0] - scores[..., -1]
        off = 4 * 65 * F32 * (query[t].double().abs().view(4, 8, 64) @ key.abs().transpose(0, 1).transpose(1, 2) / 8).amax(-1)
        clear = ((gap > 2 * off + 50) | (off < 1)).reshape(32) if key.shape[0] > 1 else torch.ones(32, dtype=torch.bool, device=out.device)
        bound = torch.where((off < 1).reshape(32, 1), bound, HALF_FP16 * exact.abs() + 2.0**-20)
        assert bool(((out[t].double() - exact).abs() <= bound)[clear].all())


# -- together, elsewhere, captured -----------------------------------------------------------
def test_a_prompt_then_tokens_as_they_are_used() -> None:
    """Two requests: prompts written and attended to, then steps; each against the values in the cache."""
    case, norms = Case(40, [0, 0], spare=12), head_norms(41)
    for row, tokens in enumerate((37, 20)):
        case.tables[row] = [case.free.pop() for _ in range(-(-tokens // 16))]
        case.lengths[row] = tokens
        positions = torch.arange(tokens, device=case.device)
        q, k, v = (randn(10 * row + i, 1, tokens, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
        rotated = int4.append_kv(case.cache, k, v, case.slots(row, 0, tokens), layer_begin=LAYER, error_flag=case.flag,
                                 positions=positions.int(), rope_table=case.rope, query=q, norms=norms)
        blocks = torch.tensor(case.tables[row], dtype=torch.int32, device=case.device)
        out = int4.prefill_attention(case.cache, LAYER, rotated[0], blocks, 0, case.flag)
        for name, got in zip(("key", "value"), int4.read_blocks(case.cache, LAYER, blocks, case.flag)):
            case.held[name][case.tables[row]] = got.double()
        for t in (0, 9, tokens - 1):
            exact, bound = attend64(rotated[0, t], *case.tokens(row, t + 1), HALF_FP16)
            assert bool(((out[t].double() - exact).abs() <= bound).all())
    for step in range(14):
        for row in range(2):
            if case.lengths[row] % 16 == 0:
                case.tables[row].append(case.free.pop())
            case.lengths[row] += 1
        q, k, v = (randn(100 + 10 * step + i, 2, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
        out = int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *case.batch(), case.flag, norms=norms)
        for row in range(2):
            blocks = torch.tensor(case.tables[row], dtype=torch.int32, device=case.device)
            for name, got in zip(("key", "value"), int4.read_blocks(case.cache, LAYER, blocks, case.flag)):
                case.held[name][case.tables[row]] = got.double()
        positions = torch.tensor(case.lengths, device=case.device) - 1
        q64 = rope64(norm64(q, norms.query[LAYER], norms.eps), case.rope, positions)
        check_rows(case, q64, out, moved=NORM_ERROR + 6 * F32 + 2.0**-22)
    assert int(case.flag.item()) == 0


def test_an_output_may_be_the_query_and_overlaps_are_read_first() -> None:
    case = Case(42, [40, 3000, 17])
    query = randn(1, 3, 32, 64).half()
    expected = int4.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    out = query.clone()
    assert torch.equal(int4.decode_attention(case.cache, LAYER, out, *case.batch(), case.flag, out), expected)
    room = torch.empty(4, 32, 64, dtype=torch.float16, device=case.device)
    room[:3] = query
    assert torch.equal(int4.decode_attention(case.cache, LAYER, room[:3], *case.batch(), case.flag, room[1:]), expected)
    fused = randn(2, 3, 40, 64).half()
    args = (case.rope, *case.batch(), case.flag)
    expected = int4.decode_layer(case.cache, LAYER, fused[:, :32], fused[:, 32:36], fused[:, 36:], *args)
    got = int4.decode_layer(case.cache, LAYER, fused[:, :32], fused[:, 32:36], fused[:, 36:], *args, fused[:, 8:])
    assert torch.equal(got, expected)


def test_rotated_queries_written_over_keys_and_values() -> None:
    """An output over K and V of other tokens, and one beside them in the same rows."""
    sides = []
    for how in ("new", "over", "beside"):
        case = Case(43, [0], spare=8)
        case.tables[0] = case.free[:4]
        fused = randn(44, 1, 50, 48, 64).half()
        query, key, value = fused[:, :, :32], fused[:, :, 32:36], fused[:, :, 36:40]
        out = {"new": torch.empty(1, 50, 32, 64, dtype=torch.float16, device=case.device), "over": fused[:, :, 8:40],
               "beside": fused[:, :, :32]}[how]
        positions = torch.arange(50, device=case.device).int()
        got = int4.append_kv(case.cache, key, value, case.slots(0, 0, 50), layer_begin=LAYER, error_flag=case.flag,
                             positions=positions, rope_table=case.rope, query=query, query_out=out)
        sides.append((got.clone(), case.cache.storage.clone()))
    for got, storage in sides[1:]:
        assert torch.equal(got, sides[0][0]) and torch.equal(storage, sides[0][1])


def test_a_cache_past_32_bits_of_offset() -> None:
    """Blocks that lie beyond 2^32 bytes in one layer."""
    blocks = 1_000_000
    cache = int4.Int4Cache.empty(1, blocks, cuda_device())
    flag = torch.zeros(1, dtype=torch.int32, device=cache.device)
    table = torch.tensor([blocks - 1, 7, blocks - 3], dtype=torch.int32, device=cache.device)
    slots = (table.long()[torch.arange(40, device=cache.device) // 16] * 16 + torch.arange(40, device=cache.device) % 16).int()
    key, value, query = randn(1, 1, 40, 4, 64).half(), randn(2, 1, 40, 4, 64).half(), randn(3, 1, 32, 64).half()
    int4.append_kv(cache, key, value, slots, layer_begin=0, error_flag=flag)
    got = int4.read_blocks(cache, 0, table, flag)
    k, v = stored(key[0].float()), stored(value[0].float())
    assert torch.equal(got[0].reshape(-1, 4, 64)[:40].double(), k) and torch.equal(got[1].reshape(-1, 4, 64)[:40].double(), v)
    as_int = lambda *x: torch.tensor(x, dtype=torch.int32, device=cache.device)  # noqa: E731
    out = int4.decode_attention(cache, 0, query, as_int(40), as_int(0, 3), table, 3, flag)
    exact, bound = attend64(query[0], k, v)
    assert bool(((out[0].double() - exact).abs() <= bound).all()) and int(flag.item()) == 0


def test_on_another_stream_and_two_at_once() -> None:
    cases = [Case(50 + i, [700, 33, 5]) for i in range(2)]
    query = randn(1, 3, 32, 64).half()
    expected = [int4.decode_attention(c.cache, LAYER, query, *c.batch(), c.flag) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    batches = [c.batch() for c in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for case, stream, batch in zip(cases, streams, batches):
            with torch.cuda.stream(stream):
                outs.append(int4.decode_attention(case.cache, LAYER, query, *batch, case.flag))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, expected[i % 2])


def test_a_captured_decode_layer_replays_on_new_inputs_beside_an_eager_one() -> None:
    case, other = Case(60, [100, 900, 31]), Case(61, [5, 64])
    query, key, value = randn(1, 3, 32, 64).half(), randn(2, 3, 4, 64).half(), randn(3, 3, 4, 64).half()
    q2, k2, v2 = randn(4, 2, 32, 64).half(), randn(5, 2, 4, 64).half(), randn(6, 2, 4, 64).half()
    batch, other_batch, norms = case.batch(), other.batch(), head_norms(7)
    call = lambda q, k, v: int4.decode_layer(case.cache, LAYER, q, k, v, case.rope, *batch, case.flag, norms=norms)  # noqa: E731
    eager = lambda: int4.decode_layer(other.cache, LAYER, q2, k2, v2, other.rope, *other_batch, other.flag)  # noqa: E731
    call(query, key, value)
    want_other = eager()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call(query, key, value)
    for seed in (11, 12):
        for tensor, at in ((query, 0), (key, 1), (value, 2)):
            tensor.copy_(randn(seed + 10 * at, *tensor.shape).half())
        graph.replay()
        assert torch.equal(eager(), want_other)
        got, storage = out.clone(), case.cache.storage.clone()
        assert torch.equal(got, call(query, key, value)) and torch.equal(storage, case.cache.storage)
    assert int(case.flag.item()) == 0


# -- refusals --------------------------------------------------------------------------------
def test_refusals() -> None:
    case = Case(70, [20])
    cache, flag, rope_table = case.cache, case.flag, case.rope
    lengths, prefix, flat, total = case.batch()
    half = lambda *shape: torch.zeros(shape, dtype=torch.float16, device=case.device)  # noqa: E731
    key, query, slots = half(1, 2, 4, 64), half(1, 32, 64), case.slots(0, 0, 2)

    def refused(match, function, *args, **kwargs):
        with pytest.raises(ValueError, match=match):
            function(*args, **kwargs)

    refused("uint8", int4.Int4Cache, cache.storage.view(torch.int8))
    refused("uint8", int4.Int4Cache, cache.storage[..., :4600])
    refused("uint8", int4.Int4Cache, cache.storage[:, ::2])
    refused("at least one", int4.Int4Cache, cache.storage[:0])
    refused("CUDA", int4.Int4Cache, cache.storage.cpu())
    refused("16-byte", int4.read_blocks, int4.Int4Cache(torch.empty(4609, dtype=torch.uint8, device=case.device)[1:].view(1, 1, 4608)),
            0, flat, flag)
    append = lambda k=key, v=key, s=slots, layer=LAYER, **kw: int4.append_kv(cache, k, v, s, layer_begin=layer, error_flag=flag, **kw)  # noqa: E731
    refused("share", append, half(1, 2, 3, 64))
    refused("share", append, v=half(1, 3, 4, 64))
    refused("FP16", append, key.float(), key.float())
    refused("FP16", append, key.cpu(), key.cpu())
    refused("slots", append, s=slots[:1])
    refused("slots", append, s=slots.long())
    refused("layers out of range", append, layer=LAYERS)
    refused("layers out of range", append, layer=-1)
    refused("layers out of range", append, half(LAYERS, 2, 4, 64), half(LAYERS, 2, 4, 64))
    refused("goes with", append, positions=slots)
    refused("goes with", append, query=half(1, 2, 32, 64))
    refused("goes with", append, query_out=half(1, 2, 32, 64))
    refused("norms go", append, norms=head_norms(1))
    both = dict(positions=slots, rope_table=rope_table)
    refused("rope_table", append, positions=slots, rope_table=rope_table[:, :100])
    refused("positions", append, positions=slots[:1], rope_table=rope_table)
    refused("query", append, query=half(1, 2, 31, 64), **both)
    refused("query_out", append, query=half(1, 2, 32, 64), query_out=half(1, 1, 32, 64).expand(1, 2, 32, 64), **both)
    refused("FP16 or FP32", append, query=half(1, 2, 32, 64), query_out=half(1, 2, 32, 64).double(), **both)
    good = head_norms(1)
    refused("head norms", append, norms=int4.HeadNorms(good.query[:1], good.key), **both)
    refused("head norms", append, norms=int4.HeadNorms(good.query, good.key.float()), **both)
    refused("head norms", append, norms=int4.HeadNorms(good.query.cpu(), good.key), **both)
    refused("eps", append, norms=int4.HeadNorms(good.query, good.key, -1.0), **both)
    refused("eps", append, norms=int4.HeadNorms(good.query, good.key, math.nan), **both)
    with pytest.raises(TypeError, match="head norms"):
        append(norms=int4.HeadNorms(None, good.key), **both)
    refused("layers out of range", int4.read_blocks, cache, LAYERS, flat, flag)
    refused("blocks", int4.read_blocks, cache, LAYER, flat.long(), flag)
    refused("error_flag", int4.read_blocks, cache, LAYER, flat, flag.cpu())
    attend = lambda q=query, n=lengths, p=prefix, f=flat, t=total, layer=LAYER, out=None: int4.decode_attention(  # noqa: E731
        cache, layer, q, n, p, f, t, flag, out)
    refused("query", attend, half(1, 32, 32))
    refused("query", attend, half(0, 32, 64))
    refused("FP16", attend, query.float())
    refused("lengths", attend, n=lengths.long())
    refused("prefix", attend, p=prefix[:1])
    refused("flat", attend, t=total + 1)
    refused("nonempty batch|total_blocks", attend, t=-1)
    refused("layers out of range", attend, layer=7)
    refused("out", attend, out=half(1, 32, 64).float())
    refused("overlap", attend, half(2, 32, 64), torch.cat((lengths, lengths)), torch.cat((prefix, prefix)),
            out=half(1, 32, 64).expand(2, 32, 64))
    layer_call = lambda k=key[0, :1], norms=None: int4.decode_layer(  # noqa: E731
        cache, LAYER, query, k, k, rope_table, lengths, prefix, flat, total, flag, norms=norms)
    refused("key", layer_call, key[0])
    refused("key", layer_call, key[0, :1].float())
    refused("head norms", layer_call, norms=int4.HeadNorms(good.query[:1], good.key))
    prompt = lambda q=query, blocks=flat, start=3: int4.prefill_attention(cache, LAYER, q, blocks, start, flag)  # noqa: E731
    refused("query", prompt, half(0, 32, 64))
    refused("below 2048", prompt, start=2048)
    refused("below 2048", prompt, start=-1)
    refused("below 2048", prompt, start=True)
    refused("blocks", prompt, start=200)
    assert int(flag.item()) == 0
