"""Strides and alignments of the 8-bit allocator's decode calls: what reaches the kernels, and the results."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8, kv_cache_fp8
from pagedcore_b200.kv_cache_fp8 import Fp8KVAllocator

ROW = 32 * 64


class Library:
    """Stands in for the native library: records what a decode layer is launched with."""

    def pkv_fp8_decode_layer(self, *args) -> int:
        names = ("query", "query_stride", "key", "value", "kv_stride")
        self.call = dict(zip(names, args[7:12])) | {"out": args[19], "out_stride": args[20]}
        return 0


@pytest.fixture
def launch(monkeypatch):
    library = Library()
    monkeypatch.setattr(kv_cache_fp8, "lib", library)
    allocator = Fp8KVAllocator.__new__(Fp8KVAllocator)
    fixed = ((0, 0, 0, 0, 22, 4), 0, 0, 0, 0, 4, 1, 0, 0, 0)

    def run(query, key, value, out):
        library.call = None
        allocator._launch_decode_layer(0, query, key, value, out, query.shape[0], fixed, 0, 0)
        return library.call

    return run


def half(*shape: int) -> torch.Tensor:
    return torch.zeros(shape, dtype=torch.float16)


def test_rows_as_they_are_reach_the_kernels_as_they_are(launch) -> None:
    wide, out = half(4, 40, 64), half(4, 48, 64)
    call = launch(wide[:, :32], wide[:, 32:36], wide[:, 36:], out[:, 8:40])
    assert call == {"query": wide.data_ptr(), "query_stride": 2560, "key": wide[:, 32:].data_ptr(),
                    "value": wide[:, 36:].data_ptr(), "kv_stride": 2560, "out": out[:, 8:].data_ptr(),
                    "out_stride": 48 * 64}
    one = half(1, ROW).expand(3, ROW)[:1].view(1, 32, 64)  # one row: any stride
    call = launch(one, half(1, 4, 64), half(1, 4, 64), one.clone())
    assert call["query"] == one.data_ptr() and call["query_stride"] == call["out_stride"] == ROW


@pytest.mark.parametrize("query", [
    half(1, 32, 64).expand(4, 32, 64),
    half(8 * ROW).as_strided((4, 32, 64), (64, 64, 1)),
    half(8 * ROW).as_strided((4, 32, 64), (ROW + 2, 64, 1)),
    half(8 * ROW)[2 : 2 + 4 * ROW].view(4, 32, 64),
], ids=["broadcast", "overlapping", "odd-stride", "unaligned"])
def test_a_query_that_the_kernels_cannot_take_is_copied(launch, query) -> None:
    call = launch(query, half(4, 4, 64), half(4, 4, 64), half(4, 32, 64))
    assert call["query"] != query.data_ptr() and call["query"] % 16 == 0 and call["query_stride"] == ROW


def test_unaligned_keys_values_and_outputs_are_copied(launch) -> None:
    base = half(8 * ROW)
    kv = base[2 : 2 + 1024].view(4, 4, 64)
    for out in (base[2 : 2 + 4 * ROW].view(4, 32, 64), base.as_strided((3, 32, 64), (ROW + 2, 64, 1))):
        rows = out.shape[0]
        call = launch(half(rows, 32, 64), kv[:rows], kv[:rows], out)
        assert call["key"] % 16 == 0 and call["value"] % 16 == 0 and call["kv_stride"] == 256
        assert call["out"] % 16 == 0 and call["out"] != out.data_ptr() and call["out_stride"] == ROW


@pytest.mark.parametrize("out", [half(1, 32, 64).expand(4, 32, 64), half(8 * ROW).as_strided((4, 32, 64), (64, 64, 1))],
                         ids=["broadcast", "overlapping"])
def test_outputs_whose_rows_overlap_are_refused(launch, out) -> None:
    with pytest.raises(ValueError, match="overlap"):
        launch(half(4, 32, 64), half(4, 4, 64), half(4, 4, 64), out)


@pytest.mark.gpu
def test_a_decode_layer_and_attention_of_any_strides_give_the_same() -> None:
    from tests.test_fp8_decoder_gpu import admit, make_allocator
    from tests.test_fp8_gpu import randn

    def step(shape):
        allocator = make_allocator(20)
        requests = admit(allocator, 3, 4, 3)
        for i, (request, n) in enumerate(zip(requests, (20, 33, 16))):
            allocator.append(request, randn(400 + i, 22, n, 4, 64).half(), randn(410 + i, 22, n, 4, 64).half(), rotate=True)
        outs = []
        with allocator.append_decode(requests):
            for layer in range(22):
                q = randn(420 + layer, 1, 32, 64).half().expand(3, 32, 64)
                k, v = (randn(450 + layer + 30 * i, 3, 4, 64).half() for i in range(2))
                arguments, out = shape(q, k, v)
                result = allocator.decode_layer(layer, *arguments, out=out)
                assert out is None or result is out
                outs.append(result.clone())
        batch = allocator.decode_batch(requests, layer_index=7)
        query, out = shape(q, k, v)[0][0], shape(q, k, v)[1]
        outs.append(allocator.attend(batch, query, layer_index=7, out=out).clone())
        allocator.check_device_errors()
        return outs

    def unaligned(tensor, gap):
        """The tensor's values in rows `gap` more than contiguous ones apart, two values off alignment."""
        rows, width = tensor.shape[0], tensor[0].numel()
        base = torch.full((rows * (width + gap) + 8,), 7.0, dtype=torch.float16, device=tensor.device)
        view = base.as_strided(tensor.shape, (width + gap, 64, 1), 2)
        return view.copy_(tensor)

    expected = step(lambda q, k, v: ((q.contiguous(), k, v), None))
    shapes = {
        "broadcast": lambda q, k, v: ((q, k, v), None),
        "unaligned": lambda q, k, v: ((unaligned(q, 0), unaligned(k, 0), unaligned(v, 0)), unaligned(torch.zeros_like(q), 0)),
        "odd": lambda q, k, v: ((unaligned(q, 2), unaligned(k, 2), unaligned(v, 2)), unaligned(torch.zeros_like(q), 2)),
        "kv": lambda q, k, v: ((q, unaligned(k, 6), v), None),
    }
    for name, shape in shapes.items():
        assert all(torch.equal(a, b) for a, b in zip(step(shape), expected)), name


@pytest.mark.gpu
def test_a_step_graph_leaves_rows_past_the_batch_alone_in_an_unaligned_output() -> None:
    from pagedcore_b200.graph import DecodeStepGraph
    from tests.test_fp8_decoder_gpu import admit, make_allocator
    from tests.test_fp8_gpu import randn

    outs = []
    for offset in (0, 2):
        allocator = make_allocator(12)
        requests = admit(allocator, 3, 3)
        for i, request in enumerate(requests):
            allocator.append(request, randn(460 + i, 22, 20, 4, 64).half(), randn(465 + i, 22, 20, 4, 64).half())
        q, k, v = (randn(470 + heads, 22, 5, heads, 64).half() for heads in (32, 4, 4))
        out = torch.full((22 * 5 * ROW + 8,), 5.0, dtype=torch.float16, device=q.device)[offset : offset + 22 * 5 * ROW]
        out = out.view(22, 5, 32, 64)
        graph = DecodeStepGraph(allocator, rows=5)
        for step in range(2):
            graph.step(q, k, v, out, requests)
            assert bool((out[:, 2:] == 5).all())
        allocator.check_device_errors()
        outs.append(out[:, :2])
    assert torch.equal(*outs)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "fp8"])
def test_a_decode_layers_output_elsewhere_is_refused(kind) -> None:
    from pagedcore_b200.kv_cache import KVAllocator
    from tests.test_fp8_decoder_gpu import admit, make_allocator
    from tests.test_fp8_gpu import randn

    if kind == "fp8":
        allocator = make_allocator(4)
    else:
        allocator = KVAllocator(torch.zeros(22, 2, 4, 16, 4, 64, dtype=torch.float16, device="cuda:0"))
    (request,) = admit(allocator, 2)
    allocator.append(request, randn(480, 22, 5, 4, 64).half(), randn(481, 22, 5, 4, 64).half())
    q, k, v = (randn(482 + heads, 1, heads, 64).half() for heads in (32, 4, 4))
    with pytest.raises(ValueError, match="out must be"):
        with allocator.append_decode((request,)):
            allocator.decode_layer(0, q, k, v, out=half(1, 32, 64))
    if kind == "fp8":
        batch = allocator.decode_batch((request,), layer_index=0)
        for out in (half(1, 32, 64), half(9 * ROW)[2 : 2 + ROW].view(1, 32, 64)):
            with pytest.raises(ValueError, match="out must be"):
                allocator.attend(batch, q, layer_index=0, out=out)
    assert allocator.cached_length(request) == 5
    allocator.check_device_errors()


@pytest.mark.gpu
def test_operators_copy_what_is_contiguous_but_not_aligned() -> None:
    from tests.test_fp8_gpu import LAYER, CacheCase, randn

    case = CacheCase(141, [40, 20])
    lengths, prefix, flat, total = case.batch()
    query = randn(142, 2, 32, 64).half()
    moved = torch.zeros(2 * ROW + 8, dtype=torch.float16, device=query.device)[4 : 4 + 2 * ROW].view(2, 32, 64).copy_(query)
    assert moved.is_contiguous() and moved.data_ptr() % 16
    expected = fp8.decode_attention(case.cache, LAYER, query, lengths, prefix, flat, total, case.flag)
    assert torch.equal(fp8.decode_attention(case.cache, LAYER, moved, lengths, prefix, flat, total, case.flag), expected)
    expected = fp8.prefill_attention(case.cache, LAYER, query, flat, 20, case.flag)
    assert torch.equal(fp8.prefill_attention(case.cache, LAYER, moved, flat, 20, case.flag), expected)
    assert int(case.flag.item()) == 0
