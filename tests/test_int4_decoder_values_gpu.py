"""The decoders and the scheduler over the 4-bit cache, held to a plain forward over what the cache holds."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from pagedcore_b200.decoder import BatchedDecoder, decode_paged, prefill_paged, prefill_paged_fused
from pagedcore_b200.decoder_fp8 import Fp8BatchedDecoder
from pagedcore_b200.dense import (
    apply_rope,
    dense_attention_fp32,
    final_logits,
    output_projection,
    project_qkv,
    rms_norm,
    swiglu,
)
from pagedcore_b200.engine_types import RequestId
from pagedcore_b200.graph import DecoderStepGraph
from pagedcore_b200.kv_cache import PrefillAppend
from pagedcore_b200.scheduler import Request, Worker
from pagedcore_b200.weights import random_weights
from tests.conftest import cuda_device
from tests.fp8_reference import F32, HALF_FP16, attend64
from tests.int4_reference import rope64, stored
from tests.test_decoder_gpu import LOGIT_TOL
from tests.test_int4_decoder_gpu import admit, assert_attends, context, make_allocator

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small():
    """22 layers of their own, with a narrow MLP and vocabulary."""
    return random_weights(5, cuda_device(), vocab=31, intermediate=32)


@pytest.fixture(scope="module")
def weights():
    return random_weights(3, cuda_device(), generator_device=cuda_device(), vocab=512)


def ids_of(seed: int, tokens: int, vocab: int = 31) -> torch.Tensor:
    device = cuda_device()
    return torch.randint(0, vocab, (1, tokens), device=device, generator=torch.Generator(device).manual_seed(seed))


@torch.inference_mode()
def plain_logits(weights, allocator, request: RequestId, ids: torch.Tensor) -> torch.Tensor:
    """Logits of ``ids`` [1, T], the last T tokens of ``request``, in plain ops; K and V are read from the cache."""
    end, tokens = allocator.cached_length(request), ids.shape[1]
    positions = torch.arange(end - tokens, end, device=ids.device)[None]
    allowed = (torch.arange(end, device=ids.device)[None] <= positions[0, :, None])[None, None]
    hidden = F.embedding(ids, weights.embedding)
    for index, layer in enumerate(weights.layers):
        query, key, _ = project_qkv(rms_norm(hidden, layer.input_norm), layer)
        query, _ = apply_rope(query, key, positions)
        key, value = (x.half().transpose(0, 1)[None] for x in context(allocator, request, index))
        hidden = hidden + output_projection(dense_attention_fp32(query, key, value, allowed), layer)
        hidden = hidden + swiglu(rms_norm(hidden, layer.post_attention_norm), layer)
    return final_logits(hidden, weights)


def close(actual: torch.Tensor, expected: torch.Tensor) -> None:
    torch.testing.assert_close(actual, expected, atol=LOGIT_TOL, rtol=LOGIT_TOL)


@pytest.mark.parametrize("how", ["fused", "batched"])
def test_prompt_logits_are_those_of_the_cached_keys_and_values(how, small) -> None:
    allocator, engine = make_allocator(12), BatchedDecoder(small)
    (request,) = admit(allocator, 8)
    for seed, tokens in ((1, 37), (2, 5), (3, 60)):  # three chunks, the last two behind a context
        ids = ids_of(seed, tokens)
        if how == "fused":
            logits = prefill_paged_fused(ids, small, allocator, request)
        else:
            logits = engine.prefill(ids, allocator, request)
        close(logits, plain_logits(small, allocator, request, ids))
    allocator.check_device_errors()


@pytest.mark.parametrize("how", ["rows", "batched", "graph"])
def test_step_logits_are_those_of_the_cached_keys_and_values(how, small) -> None:
    allocator, engine = make_allocator(20), BatchedDecoder(small)
    requests = admit(allocator, 2, 3, 6)
    for seed, (request, tokens) in enumerate(zip(requests, (1, 31, 80))):
        prefill_paged(ids_of(seed, tokens), small, allocator, request)
    graph = DecoderStepGraph(engine, allocator, rows=4) if how == "graph" else None
    for step in range(4):
        ids = ids_of(10 + step, 3).T.contiguous()
        if how == "rows":
            logits = decode_paged(ids, small, allocator, requests)
        elif how == "batched":
            logits = engine.step(ids, allocator, requests)
        else:
            logits = graph.step(ids, requests)
        for row, request in enumerate(requests):
            close(logits[row : row + 1], plain_logits(small, allocator, request, ids[row : row + 1]))
    allocator.check_device_errors()


@pytest.mark.parametrize("kind", [BatchedDecoder, Fp8BatchedDecoder], ids=["fp16", "fp8"])
def test_every_layer_gets_its_own_queries_keys_and_values(kind, weights, monkeypatch) -> None:
    """What a decoder hands over at each layer against the cache and against 64 bits, at the full sizes."""
    decoder, allocator = kind(weights), make_allocator(16)
    requests = admit(allocator, 6, 3)
    prompts, steps = [], []
    write, attend, decode = PrefillAppend.write_layer, PrefillAppend.attend, allocator.decode_layer

    def write_layer(self, layer, key, value, query, **kw):
        prompts.append([layer, key.clone(), value.clone(), query.clone()])
        return write(self, layer, key, value, query, **kw)

    def attend_layer(self, layer, query, out=None):
        result = attend(self, layer, query, out)
        prompts[-1] += [layer, query.clone(), result.clone()]
        return result

    def decode_layer(layer, query, key, value, **kw):
        steps.append([layer, query.clone(), key.clone(), value.clone()])
        steps[-1].append(decode(layer, query, key, value, **kw).clone())
        return steps[-1][-1]

    monkeypatch.setattr(PrefillAppend, "write_layer", write_layer)
    monkeypatch.setattr(PrefillAppend, "attend", attend_layer)
    monkeypatch.setattr(allocator, "decode_layer", decode_layer, raising=False)
    table, start = allocator._rope, 0
    for seed, tokens in ((1, 40), (2, 21)):
        prompts.clear()
        decoder.prefill(ids_of(seed, tokens, 512), allocator, requests[0])
        positions = torch.arange(start, start + tokens, device=table.device)
        assert [(entry[0], entry[4]) for entry in prompts] == [(layer, layer) for layer in range(22)]
        for layer, key, value, query, _, rotated, out in prompts:
            held_key, held_value = context(allocator, requests[0], layer)
            assert torch.equal(held_key[start:], stored(rope64(key, table, positions).float()))
            assert torch.equal(held_value[start:], stored(value.float()))
            exact = rope64(query, table, positions)
            size = query.double().abs() + query.double().abs().roll(32, -1)
            assert bool(((rotated.double() - exact).abs() <= 3 * F32 * size).all())
            for t in (0, tokens - 1):
                exact, bound = attend64(rotated[t], held_key[: start + t + 1], held_value[: start + t + 1], HALF_FP16)
                assert bool(((out[t].double() - exact).abs() <= bound).all())
        start += tokens
    decoder.prefill(ids_of(3, 17, 512), allocator, requests[1])
    for step in range(2):
        steps.clear()
        positions = torch.tensor([allocator.cached_length(r) for r in requests], device=table.device)
        decoder.step(torch.tensor([[3], [4 + step]], device=table.device), allocator, requests)
        assert [entry[0] for entry in steps] == list(range(22))
        for layer, query, key, value, out in steps:
            k64 = rope64(key, table, positions)
            for row, request in enumerate(requests):
                held_key, held_value = context(allocator, request, layer)
                assert torch.equal(held_key[-1], stored(k64[row].float())) and torch.equal(held_value[-1], stored(value[row].float()))
            assert_attends(allocator, requests, layer, rope64(query, table, positions), out)
    allocator.check_device_errors()


def test_the_scheduler_serves_requests_as_if_each_were_alone(small) -> None:
    """Five requests through three slots of a small pool: blocks come back and are used again."""
    wanted = [(7, 6), (33, 9), (16, 3), (50, 7), (2, 12)]  # prompt and new tokens

    def serve(chosen: list[int], blocks: int, slots: int) -> dict[str, list[int]]:
        allocator = make_allocator(blocks)

        def prefill(request: Request) -> int:
            ids = ids_of(int(request.request_id[1:]), request.prompt_tokens)
            return int(prefill_paged_fused(ids, small, allocator, request.request_id)[0, -1].argmax())

        def decode(requests) -> list[int]:
            ids = torch.tensor([[r.last_token] for r in requests], device=cuda_device())
            return decode_paged(ids, small, allocator, tuple(r.request_id for r in requests))[:, 0].argmax(-1).tolist()

        worker = Worker(allocator, prefill, decode, max_active=slots)
        for i in chosen:
            worker.submit(Request(RequestId(f"r{i}"), *wanted[i], ignore_eos=True))
        while not worker.idle():
            worker.iterate()
        allocator.check_device_errors()
        assert allocator.capacity().free_blocks == blocks
        return {str(request.request_id): request.output for request in worker.completed}

    together = serve(list(range(5)), 9, 3)
    for i, (_, new) in enumerate(wanted):
        assert len(together[f"r{i}"]) == new
        assert together[f"r{i}"] == serve([i], 5, 1)[f"r{i}"]
