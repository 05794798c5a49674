"""8-bit rows, the 8-bit linear layer and the 8-bit KV cache against 64-bit arithmetic."""

from __future__ import annotations

import math

import pytest
import torch

from pagedcore_b200 import fp8, rope
from tests.conftest import cuda_device
from tests.fp8_reference import (
    F32,
    HALF_FP16,
    CacheOracle,
    attend64,
    check_rows,
    finite_amax,
    group_amax,
    rope64,
    round_e4m3,
    scale_for,
    spread,
)

pytestmark = pytest.mark.gpu


def generator(seed: int) -> torch.Generator:
    return torch.Generator(device=cuda_device()).manual_seed(seed)


def randn(seed: int, *shape: int) -> torch.Tensor:
    return torch.randn(shape, device=cuda_device(), generator=generator(seed))


# -- rows --------------------------------------------------------------------------

# FP32 relative errors: the sum of squares (a thread adds up to 32, the tree 13
# more; halved by the root), rsqrt (2 ulp), and three products.
NORM_ERROR = 32 * F32
# exp (2 ulp), a sum, the quotient and the product.
SILU_ERROR = 8 * F32


@pytest.mark.parametrize("rows, dim", [(1, 8), (1, 2048), (3, 200), (7, 2056), (256, 2048), (2, 8192), (5, 128),
                                       (33, 64), (1030, 2048), (700, 136)])
@pytest.mark.parametrize("with_delta", [True, False])
def test_add_rms_norm(rows, dim, with_delta) -> None:
    hidden = (3 * randn(rows + dim, rows, dim)).half()
    delta = randn(rows + dim + 1, rows, dim).half() if with_delta else None
    weight = (1 + 0.1 * randn(dim, dim)).half()
    residual = torch.empty_like(hidden)
    before = hidden.clone()
    out = fp8.add_rms_norm(hidden, delta, weight, residual=residual if with_delta else None)
    assert torch.equal(hidden, before)
    total = hidden.double() + (delta.double() if with_delta else 0)
    if with_delta:
        assert torch.equal(residual, (hidden.float() + delta.float()).half())
    exact = total * torch.rsqrt(total.square().mean(1, keepdim=True) + 1e-5) * weight.double()
    check_rows(out, exact, NORM_ERROR)
    # In place: the residual is hidden itself.
    if with_delta:
        again = fp8.add_rms_norm(hidden, delta, weight)
        assert torch.equal(hidden, residual)
        assert torch.equal(again.codes.view(torch.uint8), out.codes.view(torch.uint8))


def test_add_rms_norm_rows_with_values_that_are_not_finite_stay_apart() -> None:
    hidden = randn(1, 4, 512).half()
    hidden[1, 3] = math.nan
    hidden[2, 5] = math.inf
    hidden[3] = 0
    weight = torch.ones(512, dtype=torch.float16, device=hidden.device)
    out = fp8.add_rms_norm(hidden, None, weight).to_half()
    alone = fp8.add_rms_norm(hidden[:1], None, weight).to_half()
    assert torch.equal(out[:1], alone)
    assert bool(out[1].isnan().all())
    assert bool(out[2, 5].isnan()) and not bool(out[2].isinf().any())
    assert bool((out[3] == 0).all())


@pytest.mark.parametrize("rows, width", [(1, 8), (3, 136), (5, 5632), (300, 256), (70000, 8)])
def test_quantize_rows_is_one_rounding(rows, width) -> None:
    x = (randn(width, rows, width) * torch.exp2(8 * randn(rows, rows, 1))).half()
    out = fp8.quantize_rows(x)
    exact = x.double()
    scales = scale_for(group_amax(exact))
    assert torch.equal(out.scales.double(), scales)
    values = round_e4m3(exact, spread(scales, width))
    # Every stored value is an FP16 number; what overflowed to infinity is NaN.
    assert torch.equal(out.to_half().double().nan_to_num(9e9), values.nan_to_num(9e9))


def test_quantize_rows_at_the_ends_of_the_range() -> None:
    device = cuda_device()
    rows = [
        [65504.0, 60000.0, -65504.0, 1.0],  # the largest scale: codes end at 240
        [448.0, -448.0, 0.5, 2.0**-10],
        [449.0, 448.0, 1.0, 0.0],
        [2.0**-24, -(2.0**-24), 3 * 2.0**-24, 0.0],  # FP16's smallest
        [0.0, -0.0, 0.0, 0.0],
        [math.inf, 1.0, -2.0, math.nan],
        [-math.inf, math.nan, math.inf, math.nan],
        [28672.0, 28688.0, 1.0, 3.0],  # 448 * 64, and the next number
    ]
    x = torch.zeros(len(rows), 136, dtype=torch.float16, device=device)
    x[:, 130:134] = torch.tensor(rows, dtype=torch.float16, device=device)
    out = fp8.quantize_rows(x)
    scales = scale_for(group_amax(x.double()))
    assert torch.equal(out.scales.double(), scales)
    expected = round_e4m3(x.double(), spread(scales, 136))
    assert torch.equal(out.to_half().double().nan_to_num(9e9), expected.nan_to_num(9e9))
    assert not bool(out.to_half().isinf().any())


def test_quantize_rows_takes_strided_rows() -> None:
    wide = randn(2, 9, 640).half()
    part = wide[:, 64:328]
    a, b = fp8.quantize_rows(part), fp8.quantize_rows(part.contiguous())
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    out = torch.full((9, 400), 7.0, dtype=torch.float16, device=wide.device)
    assert torch.equal(a.to_half(out[:, 8:272]), b.to_half())
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 272:] == 7).all())


@pytest.mark.parametrize("rows, inter", [(1, 5632), (64, 32), (257, 5632), (3, 200)])
def test_silu_mul(rows, inter) -> None:
    gate_up = (3 * randn(inter, rows, 2 * inter)).half()
    gate, up = gate_up.double().chunk(2, -1)
    check_rows(fp8.silu_mul(gate_up), gate / (1 + torch.exp(-gate)) * up, SILU_ERROR)


def test_rows_refusals() -> None:
    device = cuda_device()
    half = lambda *shape: torch.zeros(shape, dtype=torch.float16, device=device)  # noqa: E731
    with pytest.raises(ValueError, match="weight"):
        fp8.add_rms_norm(half(2, 64), None, half(32))
    with pytest.raises(ValueError, match="delta"):
        fp8.add_rms_norm(half(2, 64), half(1, 64), half(64))
    with pytest.raises(ValueError, match="multiple of 8"):
        fp8.add_rms_norm(half(2, 60), None, half(60))
    with pytest.raises(ValueError, match="multiple of 8"):
        fp8.add_rms_norm(half(1, 8200), None, half(8200))
    with pytest.raises(ValueError, match="contiguous"):
        fp8.add_rms_norm(half(2, 128)[:, :64], None, half(64))
    with pytest.raises(ValueError, match="16-byte"):
        fp8.quantize_rows(half(1, 72)[:, 4:68])
    with pytest.raises(ValueError, match="FP16"):
        fp8.quantize_rows(half(1, 64).float())
    with pytest.raises(ValueError, match="gate_up"):
        fp8.silu_mul(half(2, 7))
    with pytest.raises(ValueError, match="must be on"):
        fp8.add_rms_norm(half(2, 64), None, half(64).cpu())
    empty = fp8.quantize_rows(half(0, 64))
    assert empty.to_half().shape == (0, 64)


# -- linear ---------------------------------------------------------------------------


def random_operands(seed: int, rows: int, n: int, k: int):
    x = fp8.quantize_rows((randn(seed, rows, k) * torch.exp(randn(seed + 1, rows, 1))).half())
    weight = fp8.quantize_weight(0.02 * randn(seed + 2, n, k))
    # Scales of a checkpoint: any positive number.
    scales = weight.scales * (0.5 + torch.rand(weight.scales.shape, device=x.codes.device, generator=generator(seed + 3)))
    return x, fp8.Fp8Weight(weight.codes, scales.contiguous())


def linear64(x, weight):
    """The product in float64 and the bound of the kernel's error.

    Products of codes are exact.  Each of the k sums of FP32 is off by at most
    2^-23 of the summed magnitudes (truncation inside the tensor core), the
    scales' product, the scaled sum and the cluster's sums by 2^-24 each (16 in
    all at most), and FP16 rounds once.
    """
    k = x.codes.shape[1]
    xv = x.codes.double() * spread(x.scales, k)
    n = weight.codes.shape[0]
    wv = weight.codes.double() * weight.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = xv @ wv.T
    magnitude = xv.abs() @ wv.abs().T
    return y, HALF_FP16 * y.abs() + (2 * k + 16) * F32 * magnitude + 2.0**-25


@pytest.mark.parametrize(
    "rows, n, k",
    [(1, 1, 16), (1, 128, 128), (1, 2560, 2048), (2, 300, 48), (7, 33, 2048), (16, 129, 144), (17, 128, 272),
     (32, 2048, 5632), (33, 200, 400), (64, 640, 2048), (65, 129, 1040), (128, 2048, 5632), (129, 500, 272),
     (256, 2560, 2048), (257, 131, 512), (600, 300, 2048), (1000, 64, 16), (2047, 2048, 272), (700, 11264, 400),
     (1500, 8200, 1040), (385, 7000, 2064)],
)
def test_linear(rows, n, k) -> None:
    x, weight = random_operands(rows + n + k, rows, n, k)
    out = fp8.linear(x, weight)
    exact, bound = linear64(x, weight)
    assert bool(((out.double() - exact).abs() <= bound).all())
    assert torch.equal(fp8.linear(x, weight), out)  # the order of the sums is fixed


def test_linear_takes_strided_rows_and_outputs() -> None:
    x, weight = random_operands(5, 40, 77, 256)
    expected = fp8.linear(x, weight)
    wide = torch.zeros(40, 512, dtype=torch.uint8, device=expected.device)
    wide[:, 128:384] = x.codes.view(torch.uint8)
    strided = fp8.Fp8Rows(wide[:, 128:384].view(torch.float8_e4m3fn), x.scales)
    out = torch.full((40, 101), 9.0, dtype=torch.float16, device=expected.device)
    assert torch.equal(fp8.linear(strided, weight, out[:, 3:80]), expected)
    assert bool((out[:, :3] == 9).all()) and bool((out[:, 80:] == 9).all())
    assert fp8.linear(fp8.Fp8Rows(x.codes[:0], x.scales[:0]), weight).shape == (0, 77)


@pytest.mark.parametrize("n, width, first", [(8203, 8216, 8), (8203, 8216, 3), (8203, 8205, 0), (8200, 8216, 8)])
def test_linear_of_many_rows_leaves_what_lies_beside_its_output(n, width, first) -> None:
    rows = 1500  # tiles of 256 rows; 8203 columns end inside 16 bytes
    x, weight = random_operands(8, rows, n, 1040)
    expected = fp8.linear(x, weight)
    out = torch.full((rows + 40, width), 9.0, dtype=torch.float16, device=expected.device)
    fp8.linear(x, weight, out[:rows, first : first + n])
    assert torch.equal(out[:rows, first : first + n], expected)
    assert bool((out[rows:] == 9).all()) and bool((out[:, :first] == 9).all()) and bool((out[:, first + n :] == 9).all())


def test_linear_keeps_rows_apart() -> None:
    x, weight = random_operands(6, 20, 256, 384)
    clean = fp8.linear(x, weight)
    codes = x.codes.view(torch.uint8).clone()
    codes[3, 200] = 0x7F  # NaN
    scales = x.scales.clone()
    scales[5, 1] = math.inf
    out = fp8.linear(fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), scales), weight)
    keep = [row for row in range(20) if row not in (3, 5)]
    assert torch.equal(out[keep], clean[keep])
    assert bool(out[3].isnan().all()) and not bool(out[5].isfinite().any())


def test_linear_refusals() -> None:
    x, weight = random_operands(7, 4, 64, 128)
    bad = fp8.Fp8Rows(x.codes, x.scales[:, :0])
    with pytest.raises(ValueError, match="scales"):
        fp8.linear(bad, weight)
    with pytest.raises(ValueError, match=r"\[n, 128\]"):
        fp8.linear(x, fp8.Fp8Weight(weight.codes[:, :64].contiguous(), weight.scales))
    with pytest.raises(ValueError, match="weight needs"):
        fp8.linear(x, fp8.Fp8Weight(weight.codes, weight.scales.double()))
    narrow = fp8.quantize_rows(torch.zeros(4, 24, dtype=torch.float16, device=x.codes.device))
    with pytest.raises(ValueError, match="multiple of 16"):
        fp8.linear(narrow, fp8.quantize_weight(torch.zeros(8, 24, device=x.codes.device)))
    with pytest.raises(ValueError, match="out must be"):
        fp8.linear(x, weight, torch.empty(4, 63, dtype=torch.float16, device=x.codes.device))


def test_norm_linear_silu_linear_run_together() -> None:
    """One MLP as the decoder runs it: every stage within its bound of the stage before's actual values."""
    hidden = randn(11, 20, 512).half()
    delta = randn(12, 20, 512).half()
    norm = (1 + 0.1 * randn(13, 512)).half()
    up = fp8.quantize_weight(0.05 * randn(14, 2 * 768, 512))
    down = fp8.quantize_weight(0.05 * randn(15, 512, 768))
    x = fp8.add_rms_norm(hidden, delta, norm)
    gate_up = fp8.linear(x, up)
    act = fp8.silu_mul(gate_up)
    out = fp8.linear(act, down)
    for rows, weight, result in ((x, up, gate_up), (act, down, out)):
        exact, bound = linear64(rows, weight)
        assert bool(((result.double() - exact).abs() <= bound).all())
    gate, u = gate_up.double().chunk(2, -1)
    check_rows(act, gate / (1 + torch.exp(-gate)) * u, SILU_ERROR)


# -- cache ---------------------------------------------------------------------------

LAYERS, LAYER = 3, 1


class CacheCase:
    """Requests in an 8-bit cache whose unwritten storage holds NaN codes and NaN scales."""

    def __init__(self, seed: int, lengths: list[int], *, rotate: bool = False, spare: int = 2, spread: float = 0.0):
        device = cuda_device()
        self.device, self.lengths = device, lengths
        counts = [-(-n // 16) for n in lengths]
        blocks = sum(counts) + len(lengths) + spare
        self.cache = fp8.Fp8Cache.empty(LAYERS, blocks, device)
        for codes in (self.cache.key_codes, self.cache.value_codes):
            codes.view(torch.uint8).fill_(0x7F)
        for scales in (self.cache.key_scales, self.cache.value_scales):
            scales.fill_(math.nan)
        self.flag = torch.zeros(1, dtype=torch.int32, device=device)
        self.rope = rope.device_table(device)
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables, self.free = [], order
        for count in counts:
            self.tables.append([order.pop() for _ in range(count)])
        self.key, self.value = CacheOracle(blocks, device), CacheOracle(blocks, device)
        for row, length in enumerate(lengths):
            if length:
                factor = torch.exp2(spread * randn(seed + 5 * row + 3, length, 4, 1))
                self.append(row, randn(seed + 5 * row + 1, length, 4, 64) * factor, randn(seed + 5 * row + 2, length, 4, 64) * factor, 0)

    def slots(self, row: int, start: int, count: int) -> list[int]:
        return [self.tables[row][p // 16] * 16 + p % 16 for p in range(start, start + count)]

    def append(self, row: int, key: torch.Tensor, value: torch.Tensor, start: int) -> None:
        slots = self.slots(row, start, key.shape[0])
        fp8.append_kv(self.cache, key.half()[None], value.half()[None],
                      torch.tensor(slots, dtype=torch.int32, device=self.device), layer_begin=LAYER,
                      error_flag=self.flag)
        self.key.append(key.half(), slots)
        self.value.append(value.half(), slots)

    def batch(self):
        """lengths, prefix, flat on the device and the block count."""
        flat = [block for table in self.tables for block in table]
        prefix = [0]
        for table in self.tables:
            prefix.append(prefix[-1] + len(table))
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
        return as_int(self.lengths), as_int(prefix), as_int(flat), len(flat)

    def check_values(self) -> None:
        """What the cache holds at every written slot is what the oracle holds."""
        for row, length in enumerate(self.lengths):
            if not length:
                continue
            blocks = torch.tensor(self.tables[row], dtype=torch.int32, device=self.device)
            key, value = fp8.read_blocks(self.cache, LAYER, blocks, self.flag)
            assert torch.equal(key.reshape(-1, 4, 64)[:length].double(), self.key.tokens(self.tables[row], length))
            assert torch.equal(value.reshape(-1, 4, 64)[:length].double(), self.value.tokens(self.tables[row], length))
        assert int(self.flag.item()) == 0

    def check_attention(self, query: torch.Tensor, out: torch.Tensor) -> None:
        for row, length in enumerate(self.lengths):
            exact, bound = attend64(query[row], self.key.tokens(self.tables[row], length),
                                    self.value.tokens(self.tables[row], length))
            assert bool(((out[row].double() - exact).abs() <= bound).all()), (row, length)


def test_append_by_prompt_and_by_token() -> None:
    case = CacheCase(1, [40, 1, 16, 33])
    case.check_values()
    for row in range(4):
        if case.lengths[row] % 16 == 0:
            case.tables[row].append(case.free.pop())
        # Much larger values: the tile's scale is raised, its codes rounded again.
        case.append(row, 50 * randn(90 + row, 1, 4, 64), 300 * randn(95 + row, 1, 4, 64), case.lengths[row])
        case.lengths[row] += 1
    case.check_values()
    # A chunk that starts inside a block.
    case.tables[0] += [case.free.pop(), case.free.pop()]
    case.append(0, randn(77, 37, 4, 64), randn(78, 37, 4, 64), 41)
    case.lengths[0] += 37
    case.check_values()


def test_append_leaves_everything_else_as_it_was() -> None:
    case = CacheCase(2, [20, 5])
    before = [t.view(torch.uint8).clone() for t in (case.cache.key_codes, case.cache.value_codes)]
    case.append(0, 9 * randn(3, 3, 4, 64), 9 * randn(4, 3, 4, 64), 20)
    case.lengths[0] = 23
    case.check_values()
    block = case.tables[0][1]
    for old, codes, late in zip(before, (case.cache.key_codes, case.cache.value_codes), (False, True)):
        now = codes.view(torch.uint8).clone()
        free = (slice(None), slice(7, 16)) if not late else (slice(None), slice(None), slice(7, 16))
        assert torch.equal(now[LAYER, block][free], old[LAYER, block][free])  # the free slots of the block
        now[LAYER, block] = old[LAYER, block]
        assert torch.equal(now, old)  # every other block and layer


def test_append_twice_leaves_the_same_bytes_and_several_layers_at_once() -> None:
    case = CacheCase(3, [18])
    key, value = randn(5, LAYERS, 1, 4, 64).half(), randn(6, LAYERS, 1, 4, 64).half()
    slot = torch.tensor(case.slots(0, 18, 1), dtype=torch.int32, device=case.device)
    for layer in (0, 2):  # give the other layers the same history
        for t in (case.cache.key_codes, case.cache.value_codes):
            t.view(torch.uint8)[layer] = t.view(torch.uint8)[LAYER]
        for t in (case.cache.key_scales, case.cache.value_scales):
            t[layer] = t[LAYER]
    write = lambda: fp8.append_kv(case.cache, key, value, slot, layer_begin=0, error_flag=case.flag)  # noqa: E731
    write()
    state = [t.view(torch.uint8).clone() for t in (case.cache.key_codes, case.cache.value_codes)]
    write()
    assert all(torch.equal(a, t.view(torch.uint8))
               for a, t in zip(state, (case.cache.key_codes, case.cache.value_codes)))
    case.key.append(key[LAYER], [int(slot)])
    case.value.append(value[LAYER], [int(slot)])
    case.lengths[0] = 19
    case.check_values()


def test_append_stores_values_that_are_not_finite_as_nan() -> None:
    case = CacheCase(4, [3])
    key, value = randn(5, 2, 4, 64), randn(6, 2, 4, 64)
    key[0, 1, 7], value[1, 2, 9], value[0, 2, 9] = math.inf, math.nan, -math.inf
    case.append(0, key, value, 3)
    got_k, got_v = fp8.read_blocks(case.cache, LAYER, torch.tensor(case.tables[0], dtype=torch.int32, device=case.device),
                                   case.flag)
    for got, oracle in ((got_k, case.key), (got_v, case.value)):
        want = oracle.tokens(case.tables[0], 5)
        assert torch.equal(got[0, :5].double().nan_to_num(9e9), want.nan_to_num(9e9))


@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 100), (5, 3), (16, 16), (31, 50), (2040, 8)])
def test_append_rotates_once_in_fp32(start, tokens) -> None:
    case = CacheCase(6, [start], spare=8)
    table = case.tables[0]
    while len(table) * 16 < start + tokens:
        table.append(case.free.pop())
    key, value, query = randn(1, tokens, 4, 64).half(), randn(2, tokens, 4, 64).half(), randn(3, tokens, 32, 64).half()
    positions = torch.arange(start, start + tokens, device=case.device)
    wide = torch.zeros(1, tokens, 40, 64, dtype=torch.float16, device=case.device)  # a fused projection's rows
    wide[0, :, :32], wide[0, :, 32:36], wide[0, :, 36:] = query, key, value
    slots = case.slots(0, start, tokens)
    rotated = fp8.append_kv(
        case.cache, wide[:, :, 32:36], wide[:, :, 36:], torch.tensor(slots, dtype=torch.int32, device=case.device),
        layer_begin=LAYER, error_flag=case.flag, positions=positions.int(), rope_table=case.rope,
        query=wide[:, :, :32], query_out=wide[:, :, :32],
    )
    # Two products and a sum in FP32, then one FP16 rounding.
    exact = rope64(query, case.rope, positions)
    size = query.double().abs() + query.double().abs().roll(32, -1)
    assert bool(((rotated[0].double() - exact).abs() <= HALF_FP16 * exact.abs() + 3 * F32 * size + 2.0**-25).all())
    # K: the tile's scale, and half a step of E4M3 at it.
    k64 = rope64(key, case.rope, positions)
    blocks = torch.tensor(table, dtype=torch.int32, device=case.device)
    got, _ = fp8.read_blocks(case.cache, LAYER, blocks, case.flag)
    got = got.reshape(-1, 4, 64)[start : start + tokens].double()
    at = torch.tensor([table[p // 16] for p in range(start, start + tokens)], device=case.device)
    scale = case.cache.key_scales[LAYER][at].double()[..., None]
    ksize = key.double().abs() + key.double().abs().roll(32, -1)
    bound = torch.maximum(2.0**-4 * k64.abs(), scale * 2.0**-10) * (1 + 2.0**-20) + 3 * F32 * ksize
    assert bool(((got - k64).abs() <= bound).all())
    assert bool((finite_amax(got, (0, 2)) > 0).all())
    assert int(case.flag.item()) == 0


@pytest.mark.parametrize(
    "lengths",
    [[1], [15], [16], [17], [64], [65], [0], [0, 0, 5, 0], [3, 0, 200, 64, 1, 0], [2048], [100, 513, 2048, 17],
     [1] * 70, [33, 64, 1, 128, 127, 129] * 11, [0] * 40 + [700]],
    ids=lambda v: f"{len(v)}rows{max(v)}",
)
def test_decode_attention(lengths) -> None:
    case = CacheCase(sum(lengths) + len(lengths), lengths)
    query = randn(9, len(lengths), 32, 64).half()
    out = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    assert int(case.flag.item()) == 0
    case.check_attention(query, out)
    again = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    assert torch.equal(out, again)


def test_decode_attention_does_not_depend_on_the_room_of_the_block_list() -> None:
    """A launch sized for a larger batch (a captured one) cuts the list as one sized for this batch does."""
    case = CacheCase(16, [300, 5, 64])
    lengths, prefix, flat, total = case.batch()
    query = randn(3, 3, 32, 64).half()
    expected = fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total, case.flag)
    room = torch.cat((flat, torch.full((5000,), -7, dtype=torch.int32, device=case.device)))
    out = fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, room, room.numel(), case.flag)
    assert int(case.flag.item()) == 0
    assert torch.equal(out, expected)
    fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total - 1, case.flag)  # too little room
    assert int(case.flag.item()) == 1


def test_decode_attention_with_blocks_of_very_different_scale() -> None:
    """V's scale goes into the weights' exponent: tiny and huge blocks in one row lose nothing."""
    case = CacheCase(12, [300, 90], spread=4.0)
    query = 2 * randn(10, 2, 32, 64).half()
    out = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    case.check_attention(query, out)


def test_decode_attention_strides_and_rows_behind_the_last() -> None:
    case = CacheCase(13, [70, 20, 5])
    wide = randn(11, 3, 48, 64).half()
    query = wide[:, 8:40]
    out = torch.full((5, 40, 64), 3.0, dtype=torch.float16, device=case.device)
    result = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag, out[:3, :32])
    case.check_attention(query, result)
    assert bool((out[3:] == 3).all()) and bool((out[:, 32:] == 3).all())


def test_decode_attention_is_nan_only_where_the_cache_is() -> None:
    case = CacheCase(14, [40, 40])
    key = randn(1, 1, 4, 64)
    key[0, 2, 5] = math.nan
    case.append(0, key, randn(2, 1, 4, 64), 40)
    case.lengths[0] = 41
    query = randn(15, 2, 32, 64).half()
    out = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    nan = out.isnan()
    assert bool(nan[0, 16:24].all()) and not bool(nan[0, :16].any()) and not bool(nan[0, 24:].any()) and not bool(nan[1].any())


def test_a_block_outside_the_cache_sets_the_flag() -> None:
    case = CacheCase(15, [40])
    lengths, prefix, flat, total = case.batch()
    flat[1] = case.cache.num_blocks
    fp8.decode_attention(case.cache, LAYER, randn(1, 1, 32, 64).half(), lengths, prefix, flat, total, case.flag)
    assert int(case.flag.item()) == 1
    case.flag.zero_()
    fp8.read_blocks(case.cache, LAYER, flat, case.flag)
    assert int(case.flag.item()) == 1
    case.flag.zero_()
    bad = torch.tensor([-1], dtype=torch.int32, device=case.device)
    fp8.append_kv(case.cache, randn(1, 1, 1, 4, 64).half(), randn(1, 1, 1, 4, 64).half(), bad, layer_begin=0,
                  error_flag=case.flag)
    assert int(case.flag.item()) == 1


@pytest.mark.parametrize("lengths", [[1], [16, 17], [1, 15, 16, 48, 700, 65], [2048, 3]], ids=str)
def test_decode_layer_writes_as_append_does_and_attends(lengths) -> None:
    whole, parts = (CacheCase(21, [n - 1 for n in lengths]) for _ in range(2))
    for case in (whole, parts):
        for row, length in enumerate(lengths):
            if len(case.tables[row]) * 16 < length:
                case.tables[row].append(case.free.pop())
            case.lengths[row] = length
    count = len(lengths)
    fused = randn(22, count, 40, 64).half()
    query, key, value = fused[:, :32], fused[:, 32:36], fused[:, 36:]
    out = fp8.decode_layer(whole.cache, LAYER, query, key, value, whole.rope, *whole.batch(), whole.flag)
    slots = torch.tensor([parts.slots(row, n - 1, 1)[0] for row, n in enumerate(lengths)], dtype=torch.int32,
                         device=parts.device)
    positions = torch.tensor(lengths, dtype=torch.int32, device=parts.device) - 1
    fp8.append_kv(parts.cache, key[None], value[None], slots, layer_begin=LAYER, error_flag=parts.flag,
                  positions=positions, rope_table=parts.rope)
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        assert torch.equal(getattr(whole.cache, name).view(torch.uint8), getattr(parts.cache, name).view(torch.uint8))
    assert int(whole.flag.item()) == 0
    # The query is rotated in FP32 and kept as two FP16 numbers: 2^-22 of it, and the rotation's 3 roundings.
    rotated = rope64(query, whole.rope, positions.long())
    for row, length in enumerate(lengths):
        blocks = torch.tensor(whole.tables[row], dtype=torch.int32, device=whole.device)
        k, v = (t.reshape(-1, 4, 64)[:length].double() for t in fp8.read_blocks(whole.cache, LAYER, blocks, whole.flag))
        exact, bound = attend64(rotated[row], k, v)
        size = (query[row].double().abs() + query[row].double().abs().roll(32, -1)).view(4, 8, 64)
        moved = (4 * F32 + 2.0**-22) * (size @ k.transpose(0, 1).abs().transpose(1, 2) / 8).amax(-1, keepdim=True)
        bound = bound + (2 * moved * v.abs().amax(0)[:, None]).reshape(32, 64)
        assert bool(((out[row].double() - exact).abs() <= bound).all()), length


def test_decode_layer_flags_a_row_without_a_token() -> None:
    case = CacheCase(23, [0, 20])
    case.tables[0].append(case.free.pop())
    before = case.cache.key_codes.view(torch.uint8)[LAYER, case.tables[0][0]].clone()
    q, k, v = (randn(i, 2, h, 64).half() for i, h in ((1, 32), (2, 4), (3, 4)))
    fp8.decode_layer(case.cache, LAYER, q, k, v, case.rope, *case.batch(), case.flag)
    assert int(case.flag.item()) & 2
    assert torch.equal(case.cache.key_codes.view(torch.uint8)[LAYER, case.tables[0][0]], before)


@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 15), (0, 130), (7, 40), (100, 64), (601, 75), (2000, 48)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prefill_attention(start, tokens, dtype) -> None:
    case = CacheCase(31, [start + tokens])
    query = randn(32, tokens, 32, 64).to(dtype)
    blocks = case.batch()[2]
    wide = torch.full((tokens + 1, 40, 64), 3.0, dtype=torch.float16, device=case.device)
    out = fp8.prefill_attention(case.cache, LAYER, query, blocks, start, case.flag, wide[:tokens, 4:36])
    assert int(case.flag.item()) == 0
    for t in {0, 1, tokens // 2, tokens - 1} & set(range(tokens)):
        exact, bound = attend64(query[t], case.key.tokens(case.tables[0], start + t + 1),
                                case.value.tokens(case.tables[0], start + t + 1), HALF_FP16)
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t
    assert bool((wide[tokens] == 3).all()) and bool((wide[:, :4] == 3).all()) and bool((wide[:, 36:] == 3).all())
    assert torch.equal(fp8.prefill_attention(case.cache, LAYER, query, blocks, start, case.flag), out)


def test_prefill_attention_with_blocks_of_very_different_scale_and_a_bad_block() -> None:
    case = CacheCase(33, [300], spread=4.0)
    query = 2 * randn(34, 300, 32, 64).half()
    blocks = case.batch()[2].clone()
    out = fp8.prefill_attention(case.cache, LAYER, query, blocks, 0, case.flag)
    for t in (0, 17, 200, 299):
        exact, bound = attend64(query[t], case.key.tokens(case.tables[0], t + 1),
                                case.value.tokens(case.tables[0], t + 1), HALF_FP16)
        # FP16 weights end at 2^-24, the largest is 2^7 or more: half a step is 2^-32 of the largest V a token.
        bound = bound + 300 * 2.0**-32 * case.value.tokens(case.tables[0], t + 1).abs().amax()
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t
    blocks[3] = -1
    fp8.prefill_attention(case.cache, LAYER, query, blocks, 0, case.flag)
    assert int(case.flag.item()) == 1


def test_append_returns_the_query_in_fp32_for_the_prompt() -> None:
    case = CacheCase(35, [0], spare=4)
    case.tables[0] += [case.free.pop() for _ in range(3)]
    key, value, query = randn(1, 1, 40, 4, 64).half(), randn(2, 1, 40, 4, 64).half(), randn(3, 1, 40, 32, 64).half()
    positions = torch.arange(40, device=case.device)
    slots = torch.tensor(case.slots(0, 0, 40), dtype=torch.int32, device=case.device)
    rotated = fp8.append_kv(case.cache, key, value, slots, layer_begin=LAYER, error_flag=case.flag,
                            positions=positions.int(), rope_table=case.rope, query=query)
    exact = rope64(query[0], case.rope, positions)
    size = query[0].double().abs() + query[0].double().abs().roll(32, -1)
    assert rotated.dtype is torch.float32
    assert bool(((rotated[0].double() - exact).abs() <= 3 * F32 * size).all())


def test_rows_that_overlap_are_refused_or_copied() -> None:
    x = randn(1, 1, 256).half()
    rows, weight = fp8.quantize_rows(x.repeat(3, 1)), fp8.quantize_weight(randn(2, 64, 256))
    with pytest.raises(ValueError, match="overlap"):
        fp8.quantize_rows(x.expand(3, 256))
    with pytest.raises(ValueError, match="overlap"):
        fp8.linear(fp8.Fp8Rows(rows.codes[:1].expand(3, 256), rows.scales), weight)
    with pytest.raises(ValueError, match="overlap"):
        fp8.linear(rows, weight, torch.zeros(1, 64, dtype=torch.float16, device="cuda").expand(3, 64))
    with pytest.raises(ValueError, match="overlap"):
        rows.to_half(torch.zeros(1, 256, dtype=torch.float16, device="cuda").expand(3, 256))
    case = CacheCase(36, [40])
    query, blocks = randn(3, 1, 32, 64).half(), case.batch()[2]
    attend = lambda q, out=None: fp8.prefill_attention(case.cache, LAYER, q, blocks, 30, case.flag, out)  # noqa: E731
    assert torch.equal(attend(query.expand(3, 32, 64)), attend(query.repeat(3, 1, 1)))
    with pytest.raises(ValueError, match="overlap"):
        attend(query.repeat(3, 1, 1), torch.zeros(1, 32, 64, dtype=torch.float16, device="cuda").expand(3, 32, 64))


def test_a_cache_past_32_bits_of_offset() -> None:
    case = CacheCase(37, [0])
    blocks = 2**20 + 32  # 4096 bytes of K codes a block: the last ones begin past 2^32
    cache = fp8.Fp8Cache.empty(1, blocks, "cuda")
    small = fp8.Fp8Cache.empty(1, 4, "cuda")
    key, value, query = randn(1, 1, 40, 4, 64).half(), randn(2, 1, 40, 4, 64).half(), randn(3, 1, 40, 32, 64).half()
    positions, results = torch.arange(40, dtype=torch.int32, device="cuda"), []
    for pool, table in ((cache, [blocks - 1, blocks - 3, 2**19 + 1]), (small, [0, 1, 2])):
        flat = torch.tensor(table, dtype=torch.int32, device="cuda")
        slots = (flat[positions.long() // 16] * 16 + positions % 16).int()
        rotated = fp8.append_kv(pool, key[:, :39], value[:, :39], slots[:39], layer_begin=0, error_flag=case.flag,
                                positions=positions[:39], rope_table=case.rope, query=query[:, :39])
        prompt = fp8.prefill_attention(pool, 0, rotated[0], flat, 0, case.flag)
        lengths, prefix = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([40], [0, 3]))
        new = fp8.decode_layer(pool, 0, query[0, 39:], key[0, 39:], value[0, 39:], case.rope, lengths, prefix, flat, 3,
                               case.flag)
        read = [x.reshape(-1, 4, 64)[:40] for x in fp8.read_blocks(pool, 0, flat, case.flag)]
        results.append((prompt, new, *read))
    assert int(case.flag.item()) == 0
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_operators_on_another_stream_and_two_at_once() -> None:
    case = CacheCase(38, [300, 40, 17])
    lengths, prefix, flat = case.batch()[:3]
    query, x, weight = randn(39, 3, 32, 64).half(), randn(40, 70, 256).half(), fp8.quantize_weight(randn(41, 200, 256))
    total = flat.numel()
    attend = lambda: fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total, case.flag)  # noqa: E731
    product = lambda: fp8.linear(fp8.quantize_rows(x), weight)  # noqa: E731
    expected = attend(), product()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(20):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append((attend(), product()))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in results for a, b in zip(pair, expected))


def test_cache_refusals() -> None:
    case = CacheCase(41, [20])
    lengths, prefix, flat, total = case.batch()
    query = randn(1, 1, 32, 64).half()
    with pytest.raises(ValueError, match="layers out of range"):
        fp8.decode_attention(case.cache, LAYERS, query, lengths, prefix, flat, total, case.flag)
    with pytest.raises(ValueError, match="flat"):
        fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total + 1, case.flag)
    with pytest.raises(ValueError, match="prefix"):
        fp8.decode_attention(case.cache, LAYER, query, lengths, prefix[:1], flat, total, case.flag)
    with pytest.raises(ValueError, match="lengths"):
        fp8.decode_attention(case.cache, LAYER, query, lengths.long(), prefix, flat, total, case.flag)
    with pytest.raises(ValueError, match="query"):
        fp8.decode_attention(case.cache, LAYER, query.float(), lengths, prefix, flat, total, case.flag)
    with pytest.raises(ValueError, match="nonempty"):
        fp8.decode_attention(case.cache, LAYER, query[:0], lengths, prefix, flat, total, case.flag)
    with pytest.raises(ValueError, match="positions below 2048"):
        fp8.prefill_attention(case.cache, LAYER, query, flat, 2048, case.flag)
    with pytest.raises(ValueError, match="blocks"):
        fp8.prefill_attention(case.cache, LAYER, query, flat, 40, case.flag)
    with pytest.raises(ValueError, match="slots"):
        fp8.append_kv(case.cache, query[None, :, :4], query[None, :, :4], lengths[:0], layer_begin=0, error_flag=case.flag)
    with pytest.raises(ValueError, match="rope_table"):
        fp8.append_kv(case.cache, query[None, :, :4], query[None, :, :4], lengths, layer_begin=0, error_flag=case.flag,
                      positions=lengths)
    with pytest.raises(ValueError, match="scales"):
        fp8.Fp8Cache(case.cache.key_codes, case.cache.value_codes, case.cache.key_scales[:1], case.cache.value_scales)
    with pytest.raises(ValueError, match="value_codes"):
        fp8.Fp8Cache(case.cache.key_codes, case.cache.key_codes, case.cache.key_scales, case.cache.value_scales)


def test_a_captured_decode_layer_replays_on_new_inputs_beside_an_eager_one() -> None:
    lengths = [40, 100, 17]
    captured, eager = (CacheCase(51, [n - 1 for n in lengths]) for _ in range(2))
    for case in (captured, eager):
        for row, length in enumerate(lengths):
            if len(case.tables[row]) * 16 < length:
                case.tables[row].append(case.free.pop())
            case.lengths[row] = length
    tables = captured.batch()
    inputs = [randn(60 + i, 3, heads, 64).half() for i, heads in enumerate((32, 4, 4))]
    fp8.decode_plan(captured.device.index, 3, tables[3])  # sets the kernels' attributes before the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = fp8.decode_layer(captured.cache, LAYER, *inputs, captured.rope, *tables, captured.flag)
    torch.cuda.current_stream().wait_stream(side)
    for round_ in range(2):  # the second writes the same slots with other tokens
        for i, tensor in enumerate(inputs):
            tensor.copy_(randn(70 + 3 * round_ + i, *tensor.shape).half())
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            expected = fp8.decode_layer(eager.cache, LAYER, *inputs, eager.rope, *eager.batch(), eager.flag)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, expected)
    assert int(captured.flag.item()) == 0 and int(eager.flag.item()) == 0
