"""The 4-bit cache behind the allocator, and the decoders over it."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import int4
from pagedcore_b200.attention import paged_attention, paged_decode_attention
from pagedcore_b200.config import PagedCoreConfig
from pagedcore_b200.decoder import BatchedDecoder, decode_paged, prefill_paged_fused
from pagedcore_b200.decoder_fp8 import Fp8BatchedDecoder
from pagedcore_b200.engine_types import KVReservation, RequestId
from pagedcore_b200.graph import DecoderStepGraph, DecodeStepGraph
from pagedcore_b200.kv_cache_int4 import Int4KVAllocator, allocate_int4_kv_pool
from pagedcore_b200.weights import random_weights
from tests.conftest import cuda_device
from tests.fp8_reference import F32, HALF_FP16, attend64
from tests.int4_reference import norm64, rope64, scale_for, stored
from tests.test_int4_gpu import NORM_ERROR, randn

pytestmark = pytest.mark.gpu


def head_norms(seed: int) -> int4.HeadNorms:
    return int4.HeadNorms(*((1 + 0.2 * randn(seed + i, 22, 64)).half() for i in range(2)), 1e-5)


def make_allocator(blocks: int, norms: int4.HeadNorms | None = None) -> Int4KVAllocator:
    cache = int4.Int4Cache.empty(22, blocks, cuda_device())
    cache.storage.fill_(255)  # NaN wherever nothing is written
    return Int4KVAllocator(cache, norms=norms)


def admit(allocator: Int4KVAllocator, *credits: int) -> tuple[RequestId, ...]:
    requests = tuple(RequestId(f"r{i}") for i in range(len(credits)))
    for request, count in zip(requests, credits):
        allocator.create(KVReservation(request, count))
    return requests


def context(allocator: Int4KVAllocator, request: RequestId, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
    pages = list(allocator.iter_layer_blocks(request, layer_index=layer))
    return torch.cat([k for k, _ in pages]).double(), torch.cat([v for _, v in pages]).double()


def assert_attends(allocator, requests, layer: int, query: torch.Tensor, out: torch.Tensor, moved: float = 6 * F32 + 2.0**-22) -> None:
    """out [B, 32, 64] is the attention of ``query`` (FP16, or turned in 64 bits and off by ``moved``) over the cache."""
    for row, request in enumerate(requests):
        key, value = context(allocator, request, layer)
        exact, bound = attend64(query[row], key, value)
        size = query[row].double().abs().amax(-1).view(4, 8, 1)
        off = moved * size * key.abs().sum(-1).amax(0)[:, None, None] / 8
        bound = bound + (2 * off * value.abs().amax(0)[:, None]).reshape(32, 64)
        assert bool(((out[row].double() - exact).abs() <= bound).all()), (row, layer)


def test_appended_prompts_and_tokens_are_what_the_cache_holds() -> None:
    allocator = make_allocator(24)
    requests = admit(allocator, 4, 3, 5)
    lengths = [20, 33, 16]
    keys = [randn(1 + i, 22, n, 4, 64).half() for i, n in enumerate(lengths)]
    values = [randn(11 + i, 22, n, 4, 64).half() for i, n in enumerate(lengths)]
    allocator.append(requests[0], keys[0], values[0])
    allocator.append_many(requests[1:], torch.cat(keys[1:], 1), torch.cat(values[1:], 1), lengths[1:])
    step_k, step_v = randn(31, 22, 3, 4, 64).half() * 8, randn(32, 22, 3, 4, 64).half() * 8
    with allocator.append_decode(requests):
        for layer in range(22):
            if layer % 2:
                allocator.write_decode_batch(layer, step_k[layer], step_v[layer])
            else:
                for row, request in enumerate(requests):
                    allocator.write_decode_layer(request, layer, step_k[layer, row], step_v[layer, row])
    allocator.check_device_errors()
    for row, request in enumerate(requests):
        for layer in (0, 9, 21):
            for kv, (prompt, step) in enumerate(((keys, step_k), (values, step_v))):
                want = stored(torch.cat((prompt[row][layer], step[layer, row : row + 1])).float())
                assert torch.equal(context(allocator, request, layer)[kv], want)
                blocks = len(allocator.block_table(request))
                got = torch.cat([allocator.read_block(request, b)[kv][layer] for b in range(blocks)])
                assert torch.equal(got.double(), want)
    allocator.release_all(requests[0])
    assert allocator.capacity().free_blocks == 24 - 3 - 2


@pytest.mark.parametrize("normed", [False, True])
def test_decode_layers_and_the_reference_style_attention(normed) -> None:
    norms = head_norms(7) if normed else None
    allocator = make_allocator(80, norms)
    lengths = [1, 31, 600, 16]
    requests = admit(allocator, *[-(-(n + 3) // 16) for n in lengths])
    for i, (request, n) in enumerate(zip(requests, lengths)):
        key, value = randn(40 + i, 22, n, 4, 64).half(), randn(50 + i, 22, n, 4, 64).half()
        allocator.append(request, key, value, rotate=True)
        for layer in (0, 13):
            k64 = norm64(key[layer], norms.key[layer], norms.eps) if normed else key[layer]
            k64 = rope64(k64, allocator._rope, torch.arange(n, device=key.device))
            step = scale_for(k64.unflatten(-1, (4, 16)).abs().amax(-1) * (1 + 2.0**-23)).repeat_interleave(16, -1)
            assert bool(((context(allocator, request, layer)[0] - k64).abs() <= step * (0.5 + 2.0**-20)).all())
    moved = 6 * F32 + 2.0**-22 + (NORM_ERROR if normed else 0)
    for step in range(2):
        q, k, v = (randn(60 + 3 * step + i, 22, 4, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
        positions = torch.tensor([n + step for n in lengths], device=q.device)
        outs = []
        with allocator.append_decode(requests):
            for layer in range(22):
                outs.append(allocator.decode_layer(layer, q[layer], k[layer], v[layer]))
        allocator.check_device_errors()
        for layer in (0, 13):
            q64 = norm64(q[layer], norms.query[layer], norms.eps) if normed else q[layer]
            assert_attends(allocator, requests, layer, rope64(q64, allocator._rope, positions), outs[layer], moved)
    query = randn(70, 4, 32, 64).half()
    assert_attends(allocator, requests, 3, query, paged_decode_attention(query, allocator, requests, layer_index=3))
    one = paged_attention(query[2].view(1, 32, 1, 64), allocator, requests[2], layer_index=3)
    assert_attends(allocator, requests[2:3], 3, query[2:3], one.view(1, 32, 64))


@pytest.mark.parametrize("normed", [False, True])
def test_prompt_chunks_and_rotated_batches(normed) -> None:
    norms = head_norms(9) if normed else None
    allocator = make_allocator(16, norms)
    requests = admit(allocator, 6, 6)
    start = 0
    for tokens in (21, 40):
        q, k, v = (randn(10 + start + i, tokens, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
        with allocator.prefill_append(requests[0], tokens) as chunk:
            for layer in range(22):
                rotated = chunk.write_layer(layer, k, v, q)
                out = chunk.attend(layer, rotated)
            split = chunk.attend_split(layer, rotated.half())
        q64 = norm64(q, norms.query[21], norms.eps) if normed else q
        q64 = rope64(q64, allocator._rope, torch.arange(start, start + tokens, device=q.device))
        key, value = context(allocator, requests[0], 21)
        for t in (0, tokens - 1):
            exact, bound = attend64(rotated[t], key[: start + t + 1], value[: start + t + 1], HALF_FP16)
            assert bool(((out[t].double() - exact).abs() <= bound).all())
            exact, bound = attend64(rotated[t].half(), key[: start + t + 1], value[: start + t + 1])
            assert bool(((split[t].double() - exact).abs() <= bound).all())
        size = q64.abs().amax(-1, keepdim=True)
        assert bool(((rotated.double() - q64).abs() <= 2 * (NORM_ERROR + 4 * F32) * size).all())
        start += tokens
    allocator.append(requests[1], randn(3, 22, 30, 4, 64).half(), randn(4, 22, 30, 4, 64).half(), rotate=True)
    q, k, v = (randn(90 + i, 22, 2, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
    with allocator.append_decode(requests):
        for layer in range(22):
            rotated = allocator.write_decode_batch(layer, k[layer], v[layer], query=q[layer], rotate=True)
            out = allocator.attend(allocator.decode_batch(requests, layer_index=layer), rotated, layer_index=layer)
    assert_attends(allocator, requests, 21, rotated, out)
    allocator.check_device_errors()


def test_a_failed_step_or_chunk_publishes_nothing_and_touches_no_token() -> None:
    allocator = make_allocator(8)
    (request,) = admit(allocator, 5)
    allocator.append(request, randn(1, 22, 20, 4, 64).half(), randn(2, 22, 20, 4, 64).half())
    before = [context(allocator, request, layer) for layer in range(22)]
    q, k, v = (randn(i, 1, h, 64).half() for i, h in ((3, 32), (4, 4), (5, 4)))
    with pytest.raises(RuntimeError, match="boom"):
        with allocator.append_decode((request,)):
            allocator.decode_layer(0, q, k, 100 * v)
            raise RuntimeError("boom")
    with pytest.raises(RuntimeError, match="boom"):
        with allocator.prefill_append(request, 9) as chunk:
            chunk.write_layer(0, k.expand(9, 4, 64), 100 * v.expand(9, 4, 64), q.expand(9, 32, 64))
            raise RuntimeError("boom")
    assert allocator.cached_length(request) == 20
    for layer, old in enumerate(before):
        assert all(torch.equal(a, b) for a, b in zip(old, context(allocator, request, layer)))


def test_allocator_refusals_and_sizing() -> None:
    device = cuda_device()
    with pytest.raises(ValueError, match="22 layers"):
        Int4KVAllocator(int4.Int4Cache.empty(2, 4, device))
    with pytest.raises(ValueError, match="4-bit cache"):
        Int4KVAllocator(torch.zeros(22, 2, 4, 16, 4, 64, dtype=torch.float16, device=device))
    norms = head_norms(1)
    with pytest.raises(ValueError, match="head norms"):
        make_allocator(4, int4.HeadNorms(norms.query[:3], norms.key[:3]))
    with pytest.raises(ValueError, match="eps"):
        make_allocator(4, int4.HeadNorms(norms.query, norms.key, -1.0))
    pool = allocate_int4_kv_pool(PagedCoreConfig(kv_pool_mib=64, workspace_margin_mib=64))
    size = pool.storage.numel()
    assert size <= 64 * 2**20 < size + size // pool.num_blocks
    with pytest.raises(ValueError, match="CUDA device"):
        allocate_int4_kv_pool(PagedCoreConfig(kv_pool_mib=64, workspace_margin_mib=64), device="cpu")
    allocator = make_allocator(4)
    (request,) = admit(allocator, 2)
    with pytest.raises(ValueError, match="K and V must share"):
        allocator.append(request, randn(1, 22, 2, 4, 64), randn(2, 22, 2, 4, 64))
    with pytest.raises(ValueError, match="nonempty cache"):
        list(allocator.iter_layer_blocks(request, layer_index=0))
    with pytest.raises(KeyError):
        allocator.read_block(RequestId("nobody"), 0)


@pytest.mark.parametrize("rows", [6, 300])
@pytest.mark.parametrize("normed", [False, True])
def test_step_graph_serves_changing_batches(rows, normed) -> None:
    norms = head_norms(3) if normed else None
    allocator = make_allocator(120, norms)
    lengths = [5, 300, 16, 47, 900]
    requests = admit(allocator, *[-(-(n + 4) // 16) for n in lengths])
    for i, (request, n) in enumerate(zip(requests, lengths)):
        allocator.append(request, randn(80 + i, 22, n, 4, 64).half(), randn(90 + i, 22, n, 4, 64).half(), rotate=True)
    graph = DecodeStepGraph(allocator, rows=rows)
    q, k, v = (randn(100 + i, 22, rows, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
    out = torch.full((22, rows, 32, 64), 5.0, dtype=torch.float16, device=q.device)
    for step, chosen in enumerate(([0, 1, 2, 3, 4], [3, 1], [4, 0, 2])):
        batch = tuple(requests[r] for r in chosen)
        positions = torch.tensor([allocator.cached_length(r) for r in batch], device=q.device)
        out.fill_(5.0)
        graph.step(q, k, v, out, batch)
        allocator.check_device_errors()
        for layer in (0, 21):
            used = q[layer, : len(chosen)]
            q64 = rope64(norm64(used, norms.query[layer], norms.eps) if normed else used, allocator._rope, positions)
            assert_attends(allocator, batch, layer, q64, out[layer], 6 * F32 + 2.0**-22 + (NORM_ERROR if normed else 0))
        assert bool((out[:, len(chosen) :] == 5).all())  # rows past the batch
        q.copy_(randn(110 + step, *q.shape).half())
    assert graph.captures <= 2


def test_an_unaligned_output_and_one_over_the_inputs() -> None:
    sides = []
    for how in ("new", "unaligned", "over"):
        allocator = make_allocator(8)
        requests = admit(allocator, 3, 3)
        for i, request in enumerate(requests):
            allocator.append(request, randn(i, 22, 20, 4, 64).half(), randn(5 + i, 22, 20, 4, 64).half())
        fused = randn(9, 2, 40, 64).half()
        query, key, value = fused[:, :32], fused[:, 32:36], fused[:, 36:]
        out = {"new": None, "unaligned": torch.empty(2 * 2048 + 1, dtype=torch.float16, device=fused.device)[1:].view(2, 32, 64),
               "over": fused[:, 8:]}[how]
        with pytest.raises(RuntimeError, match="stop"):
            with allocator.append_decode(requests):
                sides.append(allocator.decode_layer(0, query, key, value, out=out).clone())
                raise RuntimeError("stop")
    assert torch.equal(sides[0], sides[1]) and torch.equal(sides[0], sides[2])


@pytest.fixture(scope="module")
def weights():
    return random_weights(3, cuda_device(), generator_device=cuda_device(), vocab=512)


@pytest.mark.parametrize("kind", [BatchedDecoder, Fp8BatchedDecoder], ids=["fp16", "fp8"])
def test_a_replayed_step_is_the_eager_step(kind, weights) -> None:
    """The decoders over the 4-bit cache: prompts, then steps, eager and through the step graph, bit by bit."""
    decoder = kind(weights)
    ids = torch.randint(0, 512, (1, 50), device=cuda_device(), generator=torch.Generator(cuda_device()).manual_seed(1))
    sides = []
    for graph in (False, True):
        allocator = make_allocator(16)
        requests = admit(allocator, 4, 2)
        logits = decoder.prefill(ids, allocator, requests[0])
        assert logits.shape == (1, 50, 512) and bool(logits.isfinite().all())
        decoder.prefill(ids[:, :9], allocator, requests[1])
        steps = DecoderStepGraph(decoder, allocator, rows=2) if graph else None
        token = torch.tensor([[7], [8]], device=cuda_device())
        outs = []
        for _ in range(4):
            out = steps.step(token, requests) if graph else decoder.step(token, allocator, requests)
            outs.append(out.clone())
            token = token + 1
        allocator.check_device_errors()
        assert allocator.cached_length(requests[0]) == 54
        sides.append(outs)
    for eager, replayed in zip(*sides):
        assert torch.equal(eager, replayed)


def test_the_row_decoders_run_over_the_4_bit_cache(weights) -> None:
    allocator = make_allocator(16)
    requests = admit(allocator, 4, 4)
    ids = torch.randint(0, 512, (1, 40), device=cuda_device())
    prefill_paged_fused(ids, weights, allocator, requests[0])
    BatchedDecoder(weights).prefill(ids, allocator, requests[1])
    token = torch.tensor([[5], [6]], device=cuda_device())
    rows = decode_paged(token, weights, allocator, requests)
    assert rows.shape == (2, 1, 512) and bool(rows.isfinite().all())
    allocator.check_device_errors()
    assert allocator.cached_length(requests[1]) == 41
