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
