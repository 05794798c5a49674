"""Prompt attention over the 8-bit cache: nothing but the output is rounded to FP16."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8
from pagedcore_b200.decoder import BatchedDecoder, prefill_paged_fused
from pagedcore_b200.decoder_fp8 import Fp8BatchedDecoder
from pagedcore_b200.kv_cache import PrefillAppend
from pagedcore_b200.weights import random_weights
from tests.conftest import cuda_device
from tests.fp8_reference import attend64, rope64
from tests.test_fp8_decoder_gpu import admit, make_allocator
from tests.test_fp8_gpu import LAYER, CacheCase, randn

pytestmark = pytest.mark.gpu


def check_prompt(out, query, key, value, start: int, tokens) -> None:
    """Rows ``tokens`` of a chunk at ``start`` against 64 bits over K/V [tokens, 4, 64].

    ``attend64`` with the weights as the decode kernels have them, 2^-21: an
    FP16 number and what it leaves as another.  The smallest FP16 step adds
    2^-25 a weight where the largest one is 2^7 or more: 2^-32 of the largest V.
    The kernel's own rotation (three FP32 roundings, 2^-24 each, and 2^-22 for the
    two FP16 halves, of magnitudes at most twice the rotated query's in sum: 14 in
    all) is within the 260 that ``attend64`` counts for the summed scores twice over.
    """
    for t in tokens:
        k, v = key[: start + t + 1], value[: start + t + 1]
        exact, bound = attend64(query[t], k, v)
        bound = bound + len(k) * 2.0**-32 * v.abs().amax()
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t


@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 15), (0, 130), (7, 40), (100, 64), (601, 75), (0, 2047), (2000, 48)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_attention_does_not_round_its_weights(start, tokens, dtype) -> None:
    case = CacheCase(131, [start + tokens])
    query = randn(132, tokens, 32, 64).to(dtype)
    out = fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert int(case.flag.item()) == 0
    key, value = (oracle.tokens(case.tables[0], start + tokens) for oracle in (case.key, case.value))
    check_prompt(out, query, key, value, start, sorted({0, 1, 14, tokens // 3, tokens // 2, tokens - 1} & set(range(tokens))))
    assert torch.equal(fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag), out)


class Recorded:
    """The prompt attention of an allocator's chunks: unrotated queries, outputs and where they stood."""

    def __init__(self, monkeypatch) -> None:
        self.calls = []
        write, attend = PrefillAppend.write_layer, PrefillAppend.attend

        def write_layer(chunk, layer, key, value, query, **kw):
            self.query = query.clone()
            return write(chunk, layer, key, value, query, **kw)

        def attend_layer(chunk, layer, query, out=None):
            result = attend(chunk, layer, query, out)
            self.calls.append((layer, chunk, query.dtype, self.query, result.clone()))
            return result

        monkeypatch.setattr(PrefillAppend, "write_layer", write_layer)
        monkeypatch.setattr(PrefillAppend, "attend", attend_layer)

    def check(self, allocator, layers) -> None:
        """Every recorded call at ``layers`` is the attention of the query rotated once, in 64 bits."""
        for layer, chunk, dtype, query, out in self.calls:
            if layer not in layers:
                continue
            assert dtype is torch.float32
            end = chunk.start + chunk.tokens
            key, value = (
                x.reshape(-1, 4, 64)[:end].double()
                for x in fp8.read_blocks(allocator.pool, layer, chunk.blocks, allocator._error)
            )
            rotated = rope64(query.view(chunk.tokens, 32, 64), allocator._rope, chunk.positions.long())
            check_prompt(out, rotated, key, value, chunk.start, sorted({0, 1, chunk.tokens // 2, chunk.tokens - 1} & set(range(chunk.tokens))))


def test_the_allocators_prompt_keeps_the_rotated_query_in_fp32(monkeypatch) -> None:
    recorded = Recorded(monkeypatch)
    allocator = make_allocator(16)
    (request,) = admit(allocator, 8)
    for index, tokens in enumerate((37, 1, 50)):  # the later chunks start inside a block
        with allocator.prefill_append(request, tokens) as chunk:
            for layer in range(22):
                q, k, v = (randn(200 + 30 * index + layer, tokens, heads, 64).half() for heads in (32, 4, 4))
                assert chunk.attend(layer, chunk.write_layer(layer, k, v, q)).dtype is torch.float16
        recorded.check(allocator, (0, 13, 21))
        recorded.calls.clear()
    allocator.check_device_errors()


def test_a_chunk_rotated_in_place_and_its_split_attention() -> None:
    """The caller's own choice: the query's FP16 rounding, in place; the split attention takes FP16 too."""
    allocator = make_allocator(8)
    (request,) = admit(allocator, 4)
    q, k, v = (randn(300 + heads, 33, heads, 64).half() for heads in (32, 4, 4))
    with allocator.prefill_append(request, 33) as chunk:
        for layer in range(22):
            unrounded = chunk.write_layer(layer, k, v, q)
            buffer = q.clone()
            rounded = chunk.write_layer(layer, k, v, buffer, in_place=True)
            assert rounded.data_ptr() == buffer.data_ptr() and torch.equal(rounded, unrounded.half())
            assert torch.equal(chunk.attend_split(layer, unrounded), chunk.attend_split(layer, rounded))
    allocator.check_device_errors()


@pytest.fixture(scope="module")
def weights():
    return random_weights(5, cuda_device(), generator_device=cuda_device(), vocab=512)


@pytest.mark.parametrize("kind", [BatchedDecoder, Fp8BatchedDecoder, None], ids=["fp16", "fp8", "rows"])
def test_the_decoders_prompts_keep_the_rotated_query_in_fp32(kind, weights, monkeypatch) -> None:
    recorded = Recorded(monkeypatch)
    allocator = make_allocator(8)
    (request,) = admit(allocator, 6)
    ids = torch.randint(0, 512, (1, 45), device=cuda_device(), generator=torch.Generator(cuda_device()).manual_seed(6))
    prefill = kind(weights).prefill if kind else lambda *args: prefill_paged_fused(args[0], weights, *args[1:])
    for part in (ids[:, :21], ids[:, 21:]):
        assert bool(prefill(part, allocator, request).isfinite().all())
        assert len(recorded.calls) == 22
        recorded.check(allocator, (0, 11, 21))
        recorded.calls.clear()
    allocator.check_device_errors()



def small_keys(seed: int, lengths: list[int], room: int = 0) -> CacheCase:
    """A cache whose keys are 2^-14 of the usual size: queries 2^14 times as large give ordinary scores."""
    case = CacheCase(seed, [0] * len(lengths), spare=sum(-(-(n + room) // 16) for n in lengths))
    for row, length in enumerate(lengths):
        case.tables[row] += [case.free.pop() for _ in range(-(-(length + room) // 16))]
        if length:
            case.append(row, randn(seed + 5 * row + 1, length, 4, 64) * 2.0**-14, randn(seed + 5 * row + 2, length, 4, 64), 0)
        case.lengths[row] = length
    return case


@pytest.mark.parametrize("start, tokens", [(0, 33), (100, 70), (0, 2047)])
def test_prompt_attention_takes_fp32_queries_of_any_size(start, tokens) -> None:
    """Rows from 2^-140 to 2^24, beside one another: no range of FP16 shows."""
    case = small_keys(133, [start + tokens])
    size = torch.randint(-100, 25, (tokens, 1, 1), generator=torch.Generator().manual_seed(134)).to(case.device)
    size[::2] = torch.randint(10, 20, (tokens, 1, 1), generator=torch.Generator().manual_seed(135)).to(case.device)[::2]
    query = torch.ldexp(randn(136, tokens, 32, 64), size)
    query[3] = 0.0
    query[5] = torch.ldexp(randn(137, 32, 64), torch.tensor(-140, device=query.device))  # FP32 subnormals in part
    query[7] = randn(138, 32, 64) * torch.tensor([1.0, 1e6] * 32, device=query.device)
    out = fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert int(case.flag.item()) == 0 and bool(out.isfinite().all())
    key, value = (oracle.tokens(case.tables[0], start + tokens) for oracle in (case.key, case.value))
    check_prompt(out, query, key, value, start, sorted({*range(12), *range(12, tokens, max(1, tokens // 40)), tokens - 1}))


def test_queries_that_rotate_past_fp16_stay_finite() -> None:
    """Two components near FP16's largest number rotate to up to sqrt(2) times it."""
    lengths = [1, 40, 17, 300]
    case = small_keys(139, [n - 1 for n in lengths], room=1)
    case.lengths = lengths
    query = torch.where(randn(140, 4, 32, 64) > 0, 65504.0, -65504.0).half()
    query[0] = randn(141, 32, 64).half() * 1000
    key, value = randn(142, 4, 4, 64).half() * 2.0**-14, randn(143, 4, 4, 64).half()
    exact_query = rope64(query, case.rope, torch.tensor(lengths, device=case.device) - 1)
    assert bool((exact_query[1:].abs().amax((1, 2)) > 65520).all())
    out = fp8.decode_layer(case.cache, LAYER, query, key, value, case.rope, *case.batch(), case.flag)
    assert int(case.flag.item()) == 0 and bool(out.isfinite().all())
    for row, length in enumerate(lengths):
        blocks = torch.tensor(case.tables[row], dtype=torch.int32, device=case.device)
        k, v = (x.reshape(-1, 4, 64)[:length].double() for x in fp8.read_blocks(case.cache, LAYER, blocks, case.flag))
        check_prompt(out[row : row + 1], exact_query[row : row + 1], k, v, length - 1, [0])


def test_a_prompt_that_rotates_past_fp16_stays_finite() -> None:
    case = small_keys(144, [0], room=40)
    query = torch.where(randn(145, 40, 32, 64) > 0, 65504.0, -65504.0).half()
    key, value = randn(146, 40, 4, 64).half() * 2.0**-14, randn(147, 40, 4, 64).half()
    at = torch.arange(40, device=case.device)
    slots = torch.tensor(case.slots(0, 0, 40), dtype=torch.int32, device=case.device)
    rotated = fp8.append_kv(case.cache, key[None], value[None], slots, layer_begin=LAYER, error_flag=case.flag,
                            positions=at.int(), rope_table=case.rope, query=query[None])
    blocks = torch.tensor(case.tables[0], dtype=torch.int32, device=case.device)
    out = fp8.prefill_attention(case.cache, LAYER, rotated[0], blocks, 0, case.flag)
    assert int(case.flag.item()) == 0 and bool(out.isfinite().all())
    k, v = (x.reshape(-1, 4, 64)[:40].double() for x in fp8.read_blocks(case.cache, LAYER, blocks, case.flag))
    exact_query = rope64(query, case.rope, at)
    assert float(exact_query.abs().max()) > 65520
    check_prompt(out, exact_query, k, v, 0, [0, 1, 17, 39])


def check_far(out, query, key, value) -> None:
    """``out`` [32, 64] where scores lie far apart: finite, and the value of the one that is clearly the largest."""
    assert bool(out.isfinite().all())
    scores = query.double().view(4, 8, 64) @ key.transpose(0, 1).transpose(1, 2) / 8
    weight = torch.softmax(scores, -1)
    # FP32 scores are off by some 2^-16 of their size: a lead of that and 40 more leaves the rest below 2^-40.
    lead = scores.topk(min(2, len(key)), -1).values
    clear = lead[..., 0] - lead[..., -1] > 40 + 2.0**-12 * scores.abs().amax(-1) if len(key) > 1 else lead[..., 0] == lead[..., 0]
    best = (weight @ value.transpose(0, 1)).reshape(32, 64)
    clear = clear.reshape(32)
    assert int(clear.sum()) > 16
    assert bool(((out.double() - best).abs() <= 2.0**-11 * best.abs() + 2.0**-25 + 2.0**-30 * value.abs().amax())[clear].all())


@pytest.mark.parametrize("factor", [2.0**16, 2.0**21, 2.0**25, 2.0**31, 2.0**38])
@pytest.mark.parametrize("layer_call", [False, True])
def test_decode_attention_of_scores_far_out(factor, layer_call) -> None:
    """Scores up to and past 2^24, where 1 is lost in FP32: the largest one's value, not NaN."""
    lengths = [1, 40, 17, 300, 2048]
    case = CacheCase(161, [0] * 5, spare=sum(-(-n // 16) for n in lengths))
    size = min(factor, 2.0**15)
    for row, n in enumerate(lengths):
        case.tables[row] += [case.free.pop() for _ in range(-(-n // 16))]
        case.lengths[row] = n
        key = (randn(162 + row, n, 4, 64) * (factor / size / 64 if factor > size else 1.0)).clamp(-60000, 60000)
        case.append(row, key, randn(170 + row, n, 4, 64), 0)
    query = (randn(163, 5, 32, 64) * size / 2).clamp(-65504, 65504).half()
    if layer_call:
        key, value = randn(164, 5, 4, 64).half(), randn(165, 5, 4, 64).half()
        out = fp8.decode_layer(case.cache, LAYER, query, key, value, case.rope, *case.batch(), case.flag)
        query = rope64(query, case.rope, torch.tensor(lengths, device=case.device) - 1)
    else:
        out = fp8.decode_attention(case.cache, LAYER, query, *case.batch(), case.flag)
    assert int(case.flag.item()) == 0
    for row, n in enumerate(lengths):
        blocks = torch.tensor(case.tables[row], dtype=torch.int32, device=case.device)
        k, v = (x.reshape(-1, 4, 64)[:n].double() for x in fp8.read_blocks(case.cache, LAYER, blocks, case.flag))
        check_far(out[row], query[row], k, v)


@pytest.mark.parametrize("exponent", [16, 21, 24, 25, 27, 31, 60, 100])
@pytest.mark.parametrize("start, tokens", [(0, 40), (300, 70), (0, 1300)])
def test_prompt_attention_of_scores_far_out(exponent, start, tokens) -> None:
    case = CacheCase(166, [start + tokens])
    query = torch.ldexp(randn(167, tokens, 32, 64), torch.tensor(exponent, device=case.device))
    query[1::3] *= 2.0**-exponent  # ordinary rows beside them
    out = fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert int(case.flag.item()) == 0 and bool(out.isfinite().all())
    key, value = (oracle.tokens(case.tables[0], start + tokens) for oracle in (case.key, case.value))
    check_prompt(out, query, key, value, start, range(1, tokens, 3 * max(1, tokens // 60)))
    for t in range(0, tokens, 3 * max(1, tokens // 60)):
        check_far(out[t], query[t], key[: start + t + 1], value[: start + t + 1])
