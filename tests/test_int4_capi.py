"""Refusals of the 4-bit entry points on the host, and the numbers of the 4-bit cache: no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pagedcore_b200 import _lib, int4
from tests.conftest import ROOT
from tests.int4_reference import NUMBERS, scale_for, stored

P = 0x10000  # a well-aligned address that no refused call follows
CACHE = (P, 2, 8)
lib = _lib.lib


def refused(function, *args, message: bytes) -> None:
    assert function(*args) == _lib.PKV_VALUE_ERROR
    assert message in lib.pkv_last_error(), lib.pkv_last_error()


def test_append_and_read() -> None:
    def append(cache=CACHE, begin=0, count=1, stride=256, tokens=1, rope=None, positions=None, norms=(None, None),
               query=None, query_out=None, key=P):
        return (*cache, begin, count, key, P, 0, stride, P, positions, tokens, rope, *norms, 1e-5, query, 0, 0, query_out,
                0, 0, 0, P, None)

    function = lib.pkv_int4_append_kv
    refused(function, *append(cache=(None, 2, 8)), message=b"storage")
    refused(function, *append(cache=(P + 8, 2, 8)), message=b"16-byte")
    refused(function, *append(cache=(P, 0, 8)), message=b"count out of range")
    refused(function, *append(cache=(P, 2, 1 << 28)), message=b"count out of range")
    refused(function, *append(begin=1, count=2), message=b"layers out of range")
    refused(function, *append(begin=-1), message=b"layers out of range")
    refused(function, *append(key=None), message=b"required")
    refused(function, *append(tokens=-1), message=b"required")
    refused(function, *append(key=P + 8), message=b"16-byte")
    refused(function, *append(stride=252), message=b"multiples of 8")
    refused(function, *append(rope=P), message=b"positions")
    refused(function, *append(query=P, query_out=P), message=b"positions")
    refused(function, *append(rope=P, positions=P, query=P), message=b"an output")
    refused(function, *append(norms=(P, P)), message=b"norms")
    refused(function, *append(rope=P, positions=P, norms=(P, None)), message=b"norms")
    refused(function, *append(rope=P, positions=P, norms=(P, P + 2)), message=b"16-byte")
    assert function(*append(tokens=0)) == _lib.PKV_OK  # nothing to launch
    refused(lib.pkv_int4_read_blocks, *CACHE, 2, P, 1, P, P, P, None, message=b"layers out of range")
    refused(lib.pkv_int4_read_blocks, *CACHE, 0, P, 2, P, P + 8, P, None, message=b"16-byte")
    refused(lib.pkv_int4_read_blocks, *CACHE, 0, None, 2, P, P, P, None, message=b"required")
    assert lib.pkv_int4_read_blocks(*CACHE, 0, P, 0, P, P, P, None) == _lib.PKV_OK


def test_attention() -> None:
    def decode(batch=1, total=4, grid=1, stride=2048, out=P, workspace=P, size=1 << 20, cache=CACHE, layer=0, flag=P):
        return (*cache, layer, P, stride, P, P, P, batch, total, grid, out, 2048, workspace, size, flag, None)

    function = lib.pkv_int4_decode_attention
    refused(function, *decode(batch=0), message=b"out of range")
    refused(function, *decode(total=-1), message=b"out of range")
    refused(function, *decode(grid=0), message=b"out of range")
    refused(function, *decode(stride=2040), message=b"2048 or more")
    refused(function, *decode(stride=2052), message=b"multiples of 8")
    refused(function, *decode(out=P + 8), message=b"16-byte")
    refused(function, *decode(flag=None), message=b"null pointer")
    refused(function, *decode(layer=2), message=b"layers out of range")
    refused(function, *decode(total=40, grid=4, workspace=None), message=b"workspace")
    refused(function, *decode(total=40, grid=4, size=5 * 8448 - 1), message=b"workspace")

    refused(function, *decode(batch=4, grid=3, workspace=None), message=b"workspace")  # fewer pieces than rows
    refused(function, *decode(batch=300, grid=4, workspace=None), message=b"workspace")

    def layer(key=P, kv_stride=256, rope=P, norms=(None, None)):
        return (*CACHE, 0, P, 2048, key, P, kv_stride, rope, *norms, 1e-5, P, P, P, 1, 4, 1, 1, P, 2048, None, 0, P, None)

    function = lib.pkv_int4_decode_layer
    refused(function, *layer(key=None), message=b"required")
    refused(function, *layer(rope=None), message=b"required")
    refused(function, *layer(kv_stride=250), message=b"multiples of 8")
    refused(function, *layer(norms=(P, None)), message=b"norms")
    refused(function, *layer(norms=(P, P + 2)), message=b"norms")

    def prompt(start=0, tokens=1000, stride=2048, size=63 * 16388, workspace=P):
        return (*CACHE, 0, P, 0, stride, P, start, tokens, P, 2048, workspace, size, P, None)

    function = lib.pkv_int4_prefill_attention
    refused(function, *prompt(tokens=0), message=b"positions below 2048")
    refused(function, *prompt(start=1049), message=b"positions below 2048")
    refused(function, *prompt(stride=2040), message=b"2048 or more")
    refused(function, *prompt(size=63 * 16388 - 1), message=b"workspace")
    refused(function, *prompt(workspace=None), message=b"workspace")
    refused(function, *prompt(workspace=P + 8), message=b"workspace")
    size = ctypes.c_int64()
    refused(lib.pkv_int4_prefill_plan, 0, 2040, 9, ctypes.byref(size), message=b"positions below 2048")
    refused(lib.pkv_int4_prefill_plan, 0, 0, 16, None, message=b"null pointer")
    assert lib.pkv_int4_prefill_plan(0, 0, 1000, ctypes.byref(size)) == _lib.PKV_OK and size.value == 63 * 16388
    refused(lib.pkv_int4_decode_plan, 0, 0, 4, ctypes.byref(ctypes.c_int32()), ctypes.byref(ctypes.c_int64()),
            message=b"nonempty batch")


def test_a_cache_that_is_not_on_a_gpu_is_refused() -> None:
    with pytest.raises(ValueError, match="CUDA"):
        int4.Int4Cache(torch.zeros(1, 1, int4.BLOCK_BYTES, dtype=torch.uint8))
    assert f"PKV_INT4_BLOCK_BYTES {int4.BLOCK_BYTES}\n" in (ROOT / "include" / "pagedkv.h").read_text()


def test_scale_bytes_are_fp16_numbers_and_no_value_moves_by_more_than_half_a_step() -> None:
    half = torch.arange(248, dtype=torch.int16).mul(128).view(torch.float16)
    assert half.double().tolist() == NUMBERS
    generator = torch.Generator().manual_seed(1)
    rows = (torch.randn(4000, 64, generator=generator) * torch.exp2(torch.randint(-24, 14, (4000, 1), generator=generator)))
    rows = rows.clamp(-64512, 64512).half().float()
    step = scale_for(rows.unflatten(-1, (4, 16)).abs().amax(-1)).repeat_interleave(16, -1)
    assert bool(((stored(rows) - rows.double()).abs() <= step / 2).all())
