"""Decoder steps over the 8-bit cache, every operator of a step against 64 bits where it is called."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import decoder, decoder_fp8, fp8, kernels
from pagedcore_b200.decoder import BatchedDecoder, decode_paged, prefill_paged_fused
from pagedcore_b200.decoder_fp8 import Fp8BatchedDecoder
from pagedcore_b200.graph import DecoderStepGraph
from pagedcore_b200.kv_cache_fp8 import Fp8KVAllocator
from pagedcore_b200.weights import random_weights
from tests.conftest import cuda_device
from tests.fp8_reference import attend64, check_rows, group_amax, rope64, round_e4m3, scale_for, spread
from tests.test_fp8_decoder_gpu import admit, context, make_allocator
from tests.test_fp8_gpu import NORM_ERROR, SILU_ERROR, linear64

pytestmark = pytest.mark.gpu

LENGTHS = (37, 5, 16)


@pytest.fixture(scope="module")
def weights():
    return random_weights(7, cuda_device(), generator_device=cuda_device(), vocab=512)


def ids(seed: int, count: int) -> torch.Tensor:
    return torch.randint(0, 512, (1, count), device=cuda_device(), generator=torch.Generator(cuda_device()).manual_seed(seed))


def prompts(prefill, allocator) -> tuple:
    requests = admit(allocator, *[4] * len(LENGTHS))
    for i, (request, count) in enumerate(zip(requests, LENGTHS)):
        prefill(ids(i, count), allocator, request)
    return requests


def within(out: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> None:
    exact, bound = attend64(query, key, value)
    assert bool(((out.double() - exact).abs() <= bound).all())


class CheckedLayers:
    """``Fp8KVAllocator.decode_layer`` with every row's output checked over what the cache then holds."""

    def __init__(self, monkeypatch) -> None:
        self.count = 0
        launch = Fp8KVAllocator.decode_layer

        def decode_layer(allocator, layer, query, key, value, *, out=None):
            unrotated = query.clone()
            result = launch(allocator, layer, query, key, value, out=out)
            requests = allocator._staged.requests
            positions = torch.tensor(allocator.decode_positions(), device=query.device).long()
            rotated = rope64(unrotated, allocator._rope, positions)
            for row, request in enumerate(requests):
                k, v = context(allocator, request, layer)
                assert len(k) == int(positions[row]) + 1
                within(result[row], rotated[row], k, v)
            self.count += 1
            return result

        monkeypatch.setattr(Fp8KVAllocator, "decode_layer", decode_layer)


def test_every_operator_of_an_8_bit_step_is_within_its_bound(weights, monkeypatch) -> None:
    calls = {"linear": 0, "norm": 0, "silu": 0, "rows": 0}

    class Checked:
        quantize_weight = staticmethod(fp8.quantize_weight)

        @staticmethod
        def linear(x, weight):
            out = fp8.linear(x, weight)
            exact, bound = linear64(x, weight)
            assert bool(((out.double() - exact).abs() <= bound).all())
            calls["linear"] += 1
            return out

        @staticmethod
        def add_rms_norm(hidden, delta, weight):
            total = hidden.double() + (0 if delta is None else delta.double())
            out = fp8.add_rms_norm(hidden, delta, weight)
            check_rows(out, total * torch.rsqrt(total.square().mean(1, keepdim=True) + 1e-5) * weight.double(), NORM_ERROR)
            calls["norm"] += 1
            return out

        @staticmethod
        def silu_mul(gate_up):
            gate, up = gate_up.double().chunk(2, -1)
            out = fp8.silu_mul(gate_up)
            check_rows(out, gate / (1 + torch.exp(-gate)) * up, SILU_ERROR)
            calls["silu"] += 1
            return out

        @staticmethod
        def quantize_rows(x):
            out = fp8.quantize_rows(x)
            scales = scale_for(group_amax(x.double()))
            assert torch.equal(out.scales.double(), scales)
            assert torch.equal(out.to_half().double(), round_e4m3(x.double(), spread(scales, x.shape[1])))
            calls["rows"] += 1
            return out

    kernels.linear_error_flag(cuda_device())
    kernels.check_linear_errors(cuda_device())
    layers = CheckedLayers(monkeypatch)
    model = Fp8BatchedDecoder(weights)
    monkeypatch.setattr(decoder_fp8, "fp8", Checked)
    allocator = make_allocator(16)
    requests = prompts(model.prefill, allocator)
    for step in range(2):
        assert bool(model.step(ids(10 + step, 3).view(3, 1), allocator, requests).isfinite().all())
    assert layers.count == 44
    assert calls == {"linear": 5 * 88, "norm": 5 * 44, "silu": 5 * 22, "rows": 5 * 22}
    allocator.check_device_errors()


def test_a_replayed_step_is_the_eager_step(weights) -> None:
    """The same launches over as many rows: the same bits, step after step."""
    model = Fp8BatchedDecoder(weights)
    sides = []
    for graph in (False, True):
        allocator = make_allocator(16)
        requests = prompts(model.prefill, allocator)
        steps = DecoderStepGraph(model, allocator, rows=3)
        sides.append([
            (steps.step(ids(20 + i, 3).view(3, 1), requests) if graph else model.step(ids(20 + i, 3).view(3, 1), allocator, requests)).clone()
            for i in range(4)
        ])
        allocator.check_device_errors()
    assert all(torch.equal(eager, replayed) for eager, replayed in zip(*sides))


def test_the_fp16_decoders_attention_over_the_8_bit_cache(weights, monkeypatch) -> None:
    layers = CheckedLayers(monkeypatch)
    allocator = make_allocator(16)
    requests = prompts(BatchedDecoder(weights).prefill, allocator)
    BatchedDecoder(weights).step(ids(30, 3).view(3, 1), allocator, requests)
    assert layers.count == 22

    attend, rows = decoder.paged_attention, []

    def paged_attention(query, allocator, request, *, layer_index, **kw):
        out = attend(query, allocator, request, layer_index=layer_index, **kw)
        within(out.view(32, 64), query.view(32, 64), *context(allocator, request, layer_index))
        rows.append(layer_index)
        return out

    monkeypatch.setattr(decoder, "paged_attention", paged_attention)
    decode_paged(ids(31, 3).view(3, 1), weights, allocator, requests)
    assert sorted(rows) == sorted(list(range(22)) * 3)
    allocator.check_device_errors()
    other = make_allocator(16)
    again = prompts(lambda part, side, request: prefill_paged_fused(part, weights, side, request), other)
    assert bool(decode_paged(ids(31, 3).view(3, 1), weights, other, again).isfinite().all())
    other.check_device_errors()
