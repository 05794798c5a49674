"""The 8-bit cache behind the allocator, and the 8-bit decoder over it."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import decoder_fp8, fp8
from pagedcore_b200.attention import paged_attention, paged_decode_attention
from pagedcore_b200.config import PagedCoreConfig
from pagedcore_b200.decoder import BatchedDecoder, decode_paged, prefill_paged_fused
from pagedcore_b200.decoder_fp8 import Fp8BatchedDecoder
from pagedcore_b200.engine_types import KVReservation, RequestId
from pagedcore_b200.graph import DecoderStepGraph, DecodeStepGraph
from pagedcore_b200.kv_cache_fp8 import Fp8KVAllocator, allocate_fp8_kv_pool
from pagedcore_b200.weights import random_weights
from tests.conftest import cuda_device
from tests.fp8_reference import CacheOracle, attend64, check_rows, rope64
from tests.test_fp8_gpu import NORM_ERROR, SILU_ERROR, linear64, randn

pytestmark = pytest.mark.gpu


def make_allocator(blocks: int) -> Fp8KVAllocator:
    cache = fp8.Fp8Cache.empty(22, blocks, cuda_device())
    for codes in (cache.key_codes, cache.value_codes):
        codes.view(torch.uint8).fill_(0x7F)
    for scales in (cache.key_scales, cache.value_scales):
        scales.fill_(float("nan"))
    return Fp8KVAllocator(cache)


def admit(allocator: Fp8KVAllocator, *credits: int) -> tuple[RequestId, ...]:
    requests = tuple(RequestId(f"r{i}") for i in range(len(credits)))
    for request, count in zip(requests, credits):
        allocator.create(KVReservation(request, count))
    return requests


def context(allocator: Fp8KVAllocator, request: RequestId, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
    pages = list(allocator.iter_layer_blocks(request, layer_index=layer))
    return torch.cat([k for k, _ in pages]).double(), torch.cat([v for _, v in pages]).double()


def assert_attends(allocator, requests, layer: int, query: torch.Tensor, out: torch.Tensor) -> None:
    """out [B, 32, 64] is the attention of ``query`` (FP16, or rotated in 64 bits) over what the cache holds."""
    for row, request in enumerate(requests):
        key, value = context(allocator, request, layer)
        exact, bound = attend64(query[row], key, value)
        # The kernel's rotation: three FP32 roundings and two FP16 halves, of magnitudes at most sqrt(2) of the query's.
        q, k = query[row].double().abs().amax(-1, keepdim=True).expand(32, 64).reshape(4, 8, 64), key.transpose(0, 1)
        moved = 2 * 2.0**-20 * (q @ k.abs().transpose(1, 2) / 8).amax(-1, keepdim=True)
        bound = bound + (moved * value.abs().amax(0)[:, None]).reshape(32, 64)
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
        table, length = list(allocator.block_table(request)), lengths[row] + 1
        for layer in (0, 9, 21):
            for kv, (prompt, step) in enumerate(((keys, step_k), (values, step_v))):
                oracle = CacheOracle(24, cuda_device())
                slots = [table[p // 16] * 16 + p % 16 for p in range(length)]
                oracle.append(prompt[row][layer], slots[:-1])
                oracle.append(step[layer, row : row + 1], slots[-1:])
                want = oracle.tokens(table, length)
                assert torch.equal(context(allocator, request, layer)[kv], want)
                got = torch.cat([allocator.read_block(request, b)[kv][layer] for b in range(len(table))])
                assert torch.equal(got.double(), want)
    allocator.release_all(requests[0])
    assert allocator.capacity().free_blocks == 24 - 3 - 2


def test_decode_layers_and_the_reference_style_attention() -> None:
    allocator = make_allocator(80)
    lengths = [1, 31, 600, 16]
    requests = admit(allocator, *[-(-(n + 3) // 16) for n in lengths])
    for i, (request, n) in enumerate(zip(requests, lengths)):
        allocator.append(request, randn(40 + i, 22, n, 4, 64).half(), randn(50 + i, 22, n, 4, 64).half(), rotate=True)
    for step in range(2):
        q, k, v = (randn(60 + 3 * step + i, 22, 4, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
        positions = torch.tensor([n + step for n in lengths], device=q.device)
        outs = []
        with allocator.append_decode(requests):
            for layer in range(22):
                outs.append(allocator.decode_layer(layer, q[layer], k[layer], v[layer]))
        allocator.check_device_errors()
        for layer in (0, 13):
            assert_attends(allocator, requests, layer, rope64(q[layer], allocator._rope, positions), outs[layer])
    query = randn(70, 4, 32, 64).half()
    batch = paged_decode_attention(query, allocator, requests, layer_index=3)
    assert_attends(allocator, requests, 3, query, batch)
    one = paged_attention(query[2].view(1, 32, 1, 64), allocator, requests[2], layer_index=3)
    assert_attends(allocator, requests[2:3], 3, query[2:3], one.view(1, 32, 64))


def test_a_failed_step_publishes_nothing() -> None:
    allocator = make_allocator(8)
    (request,) = admit(allocator, 3)
    allocator.append(request, randn(1, 22, 20, 4, 64).half(), randn(2, 22, 20, 4, 64).half())
    before = context(allocator, request, 5)
    with pytest.raises(RuntimeError, match="boom"):
        with allocator.append_decode((request,)):
            allocator.decode_layer(0, *(randn(i, 1, h, 64).half() for i, h in ((3, 32), (4, 4), (5, 4))))
            raise RuntimeError("boom")
    assert allocator.cached_length(request) == 20
    after = context(allocator, request, 5)
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_allocator_refusals_and_sizing() -> None:
    device = cuda_device()
    with pytest.raises(ValueError, match="22 layers"):
        Fp8KVAllocator(fp8.Fp8Cache.empty(2, 4, device))
    with pytest.raises(ValueError, match="8-bit cache"):
        Fp8KVAllocator(torch.zeros(22, 2, 4, 16, 4, 64, dtype=torch.float16, device=device))
    pool = allocate_fp8_kv_pool(PagedCoreConfig(kv_pool_mib=64, workspace_margin_mib=64))
    size = sum(t.numel() * t.element_size() for t in (pool.key_codes, pool.value_codes, pool.key_scales, pool.value_scales))
    assert size <= 64 * 2**20 < size + size // pool.num_blocks
    allocator = make_allocator(4)
    (request,) = admit(allocator, 2)
    with pytest.raises(ValueError, match="K and V must share"):
        allocator.append(request, randn(1, 22, 2, 4, 64), randn(2, 22, 2, 4, 64))
    with pytest.raises(ValueError, match="nonempty cache"):
        list(allocator.iter_layer_blocks(request, layer_index=0))
    with pytest.raises(KeyError):
        allocator.read_block(RequestId("nobody"), 0)


def test_step_graph_serves_changing_batches() -> None:
    allocator = make_allocator(120)
    lengths = [5, 300, 16, 47, 900]
    requests = admit(allocator, *[-(-(n + 4) // 16) for n in lengths])
    for i, (request, n) in enumerate(zip(requests, lengths)):
        allocator.append(request, randn(80 + i, 22, n, 4, 64).half(), randn(90 + i, 22, n, 4, 64).half(), rotate=True)
    graph = DecodeStepGraph(allocator, rows=6)
    q, k, v = (randn(100 + i, 22, 6, heads, 64).half() for i, heads in enumerate((32, 4, 4)))
    out = torch.full((22, 6, 32, 64), 5.0, dtype=torch.float16, device=q.device)
    for step, rows in enumerate(([0, 1, 2, 3, 4], [3, 1], [4, 0, 2])):
        batch = tuple(requests[r] for r in rows)
        positions = torch.tensor([allocator.cached_length(r) for r in batch], device=q.device)
        out.fill_(5.0)
        graph.step(q, k, v, out, batch)
        allocator.check_device_errors()
        for layer in (0, 21):
            assert_attends(allocator, batch, layer, rope64(q[layer, : len(rows)], allocator._rope, positions), out[layer])
        assert bool((out[:, len(rows) :] == 5).all())  # rows past the batch
        q.copy_(randn(110 + step, *q.shape).half())
    assert graph.captures <= 2


@pytest.fixture(scope="module")
def weights():
    return random_weights(3, cuda_device(), generator_device=cuda_device(), vocab=512)


def test_every_operator_of_a_decoder_step_is_within_its_bound(weights, monkeypatch) -> None:
    """A prompt and a decode step of the 8-bit decoder over the 8-bit cache, each operator checked where it is called."""
    calls = {"linear": 0, "norm": 0, "silu": 0}

    class Checked:
        quantize_rows, quantize_weight = staticmethod(fp8.quantize_rows), staticmethod(fp8.quantize_weight)

        @staticmethod
        def linear(x, weight):
            out = fp8.linear(x, weight)
            if calls["linear"] % 7 == 0:
                exact, bound = linear64(x, weight)
                assert bool(((out.double() - exact).abs() <= bound).all())
            calls["linear"] += 1
            return out

        @staticmethod
        def add_rms_norm(hidden, delta, weight):
            total = hidden.double() + (0 if delta is None else delta.double())
            out = fp8.add_rms_norm(hidden, delta, weight)
            exact = total * torch.rsqrt(total.square().mean(1, keepdim=True) + 1e-5) * weight.double()
            check_rows(out, exact, NORM_ERROR)
            calls["norm"] += 1
            return out

        @staticmethod
        def silu_mul(gate_up):
            gate, up = gate_up.double().chunk(2, -1)
            out = fp8.silu_mul(gate_up)
            check_rows(out, gate / (1 + torch.exp(-gate)) * up, SILU_ERROR)
            calls["silu"] += 1
            return out

    decoder = Fp8BatchedDecoder(weights)
    allocator = make_allocator(12)
    requests = admit(allocator, 4, 4)
    monkeypatch.setattr(decoder_fp8, "fp8", Checked)
    ids = torch.randint(0, 512, (1, 37), device=cuda_device())
    logits = decoder.prefill(ids, allocator, requests[0])
    assert logits.shape == (1, 37, 512) and bool(logits.isfinite().all())
    decoder.prefill(ids[:, :5], allocator, requests[1])
    step = decoder.step(torch.tensor([[3], [4]], device=cuda_device()), allocator, requests)
    assert step.shape == (2, 1, 512) and bool(step.isfinite().all())
    assert calls == {"linear": 3 * 88, "norm": 3 * 44, "silu": 3 * 22}
    allocator.check_device_errors()
    assert allocator.cached_length(requests[0]) == 38


def relative(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_decoder_step_graph_and_eager_step_agree(weights) -> None:
    """Both round every quantised vector to within half a step (2^-4) of the same value: they differ by a step at most."""
    decoder = Fp8BatchedDecoder(weights)
    sides = []
    ids = torch.randint(0, 512, (1, 50), device=cuda_device(), generator=torch.Generator(cuda_device()).manual_seed(1))
    for graph in (False, True):
        allocator = make_allocator(16)
        requests = admit(allocator, 4, 2)
        decoder.prefill(ids, allocator, requests[0])
        decoder.prefill(ids[:, :9], allocator, requests[1])
        steps = DecoderStepGraph(decoder, allocator, rows=4) if graph else None
        token = torch.tensor([[7], [8]], device=cuda_device())
        outs = []
        for _ in range(4):
            outs.append(steps.step(token, requests) if graph else decoder.step(token, allocator, requests))
            token = token + 1
        allocator.check_device_errors()
        sides.append(outs)
    for eager, replayed in zip(*sides):
        assert relative(replayed, eager) <= 2.0**-3


def test_the_fp16_decoders_run_over_the_8_bit_cache(weights) -> None:
    allocator = make_allocator(16)
    requests = admit(allocator, 4, 4)
    ids = torch.randint(0, 512, (1, 40), device=cuda_device())
    prefill_paged_fused(ids, weights, allocator, requests[0])
    BatchedDecoder(weights).prefill(ids, allocator, requests[1])
    token = torch.tensor([[5], [6]], device=cuda_device())
    rows = decode_paged(token, weights, allocator, requests)
    assert rows.shape == (2, 1, 512) and bool(rows.isfinite().all())
    batch = BatchedDecoder(weights).step(token, allocator, requests)
    assert batch.shape == (2, 1, 512) and bool(batch.isfinite().all())
    allocator.check_device_errors()
    assert allocator.cached_length(requests[1]) == 42
