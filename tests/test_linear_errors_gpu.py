"""The linear layers' device error flag reaches the caller: read, raised and cleared."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8, kernels
from pagedcore_b200._lib import DEVICE_BAD_BLOCK, DEVICE_WAIT_TIMEOUT
from pagedcore_b200.kv_cache import KVAllocator
from tests.conftest import cuda_device
from tests.test_fp8_decoder_gpu import make_allocator
from tests.test_fp8_gpu import linear64, random_operands

pytestmark = pytest.mark.gpu


@pytest.fixture
def flag():
    flag = kernels.linear_error_flag(cuda_device())
    kernels.check_linear_errors(cuda_device())
    yield flag
    flag.zero_()


def test_a_linear_layer_that_gave_up_is_reported_once(flag) -> None:
    flag.fill_(DEVICE_WAIT_TIMEOUT)  # as a kernel whose wait ran out leaves it
    with pytest.raises(RuntimeError, match="linear kernel reported: a bounded pipeline wait timed out"):
        kernels.check_linear_errors(cuda_device())
    kernels.check_linear_errors(cuda_device())
    assert int(flag.item()) == 0


@pytest.mark.parametrize("kind", ["fp16", "fp8"])
def test_the_allocators_check_reads_it_too(kind, flag) -> None:
    if kind == "fp8":
        allocator = make_allocator(2)
    else:
        allocator = KVAllocator(torch.zeros(22, 2, 2, 16, 4, 64, dtype=torch.float16, device=cuda_device()))
    allocator.check_device_errors()
    flag.fill_(DEVICE_WAIT_TIMEOUT)
    with pytest.raises(RuntimeError, match="linear kernel reported: a bounded pipeline wait timed out"):
        allocator.check_device_errors()
    allocator.check_device_errors()
    allocator._error.fill_(DEVICE_BAD_BLOCK)
    with pytest.raises(RuntimeError, match="physical KV block outside the pool"):
        allocator.check_device_errors()
    allocator.check_device_errors()
    assert int(flag.item()) == 0 and int(allocator._error.item()) == 0


@pytest.mark.parametrize("rows, n, k", [(1, 2560, 2048), (32, 2048, 5632), (64, 129, 144), (100, 2048, 5632), (256, 2560, 2048),
                                        (600, 300, 2048), (1500, 8200, 1040)])
def test_the_8_bit_linear_kernels_leave_it_clear(rows, n, k, flag) -> None:
    x, weight = random_operands(rows + n, rows, n, k)
    out = fp8.linear(x, weight)
    exact, bound = linear64(x, weight)
    assert bool(((out.double() - exact).abs() <= bound).all())
    kernels.check_linear_errors(cuda_device())


def test_a_flag_first_asked_for_in_a_capture_is_the_graphs_own(flag, monkeypatch) -> None:
    x, weight = random_operands(3, 20, 256, 384)
    expected = fp8.linear(x, weight)
    monkeypatch.setattr(kernels, "_linear_errors", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8.linear(x, weight)
    assert kernels.device_linear_flag(cuda_device()) is None
    kernels.check_linear_errors(cuda_device())  # nothing to read, whatever the graph's memory holds before it runs
    graph.replay()
    assert torch.equal(out, expected)
    assert torch.equal(fp8.linear(x, weight), expected) and kernels.device_linear_flag(cuda_device()) is not None
