"""Refusals of the 8-bit entry points on the host: nothing is launched, no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pagedcore_b200 import _lib, fp8
from tests.fp8_reference import round_e4m3, scale_for

P = 0x10000  # a well-aligned address that no refused call follows
CACHE = (P, P, P, P, 2, 8)
lib = _lib.lib


def refused(function, *args, message: bytes) -> None:
    assert function(*args) == _lib.PKV_VALUE_ERROR
    assert message in lib.pkv_last_error(), lib.pkv_last_error()


def test_rows() -> None:
    refused(lib.pkv_fp8_add_rms_norm, None, None, P, None, P, P, 1, 64, 1e-5, None, message=b"required")
    refused(lib.pkv_fp8_add_rms_norm, P, P, P, None, P, P, 1, 64, 1e-5, None, message=b"residual")
    refused(lib.pkv_fp8_add_rms_norm, P, None, P, None, P, P, 1, 60, 1e-5, None, message=b"multiple of 8")
    refused(lib.pkv_fp8_add_rms_norm, P, None, P, None, P, P, 1, 8200, 1e-5, None, message=b"multiple of 8")
    refused(lib.pkv_fp8_add_rms_norm, P + 2, None, P, None, P, P, 1, 64, 1e-5, None, message=b"aligned")
    refused(lib.pkv_fp8_quantize, P, 64, 1, 1, 64, P, P, None, message=b"row stride")
    refused(lib.pkv_fp8_quantize, P, 68, 0, 1, 64, P, P, None, message=b"row stride")
    refused(lib.pkv_fp8_to_half, P, P, 1, 12, P, 16, None, message=b"multiple of 8")
    refused(lib.pkv_fp8_to_half, P, P, -1, 16, P, 16, None, message=b"multiple of 8")
    assert lib.pkv_fp8_quantize(P, 64, 0, 0, 64, P, P, None) == _lib.PKV_OK  # no rows, no launch


def test_linear() -> None:
    def call(**kw):
        a = dict(x=P, stride=64, sx=P, w=P, sw=P, rows=1, n=8, k=64, out=P, out_stride=8, flag=P) | kw
        return (a["x"], a["stride"], a["sx"], a["w"], a["sw"], a["rows"], a["n"], a["k"], a["out"], a["out_stride"],
                a["flag"], None)

    refused(lib.pkv_fp8_linear, *call(sw=None), message=b"null pointer")
    refused(lib.pkv_fp8_linear, *call(k=24), message=b"multiple of 16")
    refused(lib.pkv_fp8_linear, *call(k=0), message=b"multiple of 16")
    refused(lib.pkv_fp8_linear, *call(n=0), message=b"n at least 1")
    refused(lib.pkv_fp8_linear, *call(rows=-1), message=b"multiple of 16")
    refused(lib.pkv_fp8_linear, *call(stride=72), message=b"misaligned")
    refused(lib.pkv_fp8_linear, *call(stride=48), message=b"misaligned")
    refused(lib.pkv_fp8_linear, *call(w=P + 8), message=b"misaligned")
    refused(lib.pkv_fp8_linear, *call(out_stride=7), message=b"misaligned")
    assert lib.pkv_fp8_linear(*call(rows=0)) == _lib.PKV_OK


def test_cache() -> None:
    def append(cache=CACHE, begin=0, count=1, stride=256, rope=None, positions=None, query=None, query_out=None):
        return (*cache, begin, count, P, P, 0, stride, P, positions, 1, rope, query, 0, 0, query_out, 0, 0, 0, P, None)

    refused(lib.pkv_fp8_append_kv, *append(cache=(P, None, P, P, 2, 8)), message=b"codes and scales")
    refused(lib.pkv_fp8_append_kv, *append(cache=(P + 8, P, P, P, 2, 8)), message=b"16-byte")
    refused(lib.pkv_fp8_append_kv, *append(cache=(P, P, P, P, 0, 8)), message=b"count out of range")
    refused(lib.pkv_fp8_append_kv, *append(cache=(P, P, P, P, 2, 1 << 28)), message=b"count out of range")
    refused(lib.pkv_fp8_append_kv, *append(begin=1, count=2), message=b"layers out of range")
    refused(lib.pkv_fp8_append_kv, *append(begin=-1), message=b"layers out of range")
    refused(lib.pkv_fp8_append_kv, *append(stride=252), message=b"multiples of 8")
    refused(lib.pkv_fp8_append_kv, *append(rope=P), message=b"positions")
    refused(lib.pkv_fp8_append_kv, *append(query=P, query_out=P), message=b"positions")
    refused(lib.pkv_fp8_append_kv, *append(rope=P, positions=P, query=P), message=b"an output")
    refused(lib.pkv_fp8_read_blocks, *CACHE, 2, P, 1, P, P, P, None, message=b"layers out of range")
    refused(lib.pkv_fp8_read_blocks, *CACHE, 0, P, 2, P, P + 8, P, None, message=b"16-byte")


def test_attention() -> None:
    def decode(batch=1, total=4, grid=1, stride=2048, workspace=P, size=1 << 20, cache=CACHE, layer=0):
        return (*cache, layer, P, stride, P, P, P, batch, total, grid, P, 2048, workspace, size, P, None)

    refused(lib.pkv_fp8_decode_attention, *decode(batch=0), message=b"out of range")
    refused(lib.pkv_fp8_decode_attention, *decode(total=-1), message=b"out of range")
    refused(lib.pkv_fp8_decode_attention, *decode(grid=0), message=b"out of range")
    refused(lib.pkv_fp8_decode_attention, *decode(stride=2040), message=b"2048 or more")
    refused(lib.pkv_fp8_decode_attention, *decode(workspace=None), message=b"workspace")
    refused(lib.pkv_fp8_decode_attention, *decode(grid=4, size=4096), message=b"workspace")
    refused(lib.pkv_fp8_decode_attention, *decode(layer=2), message=b"layers out of range")
    refused(lib.pkv_fp8_decode_layer, *CACHE, 0, P, 2048, None, P, 256, P, P, P, P, 1, 4, 1, P, 2048, P, 1 << 20, P, None,
            message=b"key, value and rope_table")
    def prefill(layer=0, fp32=0, stride=2048, blocks=P, start=0, tokens=17, bytes=1 << 24):
        return (*CACHE, layer, P, fp32, stride, blocks, start, tokens, P, 2048, P, bytes, P, None)

    refused(lib.pkv_fp8_prefill_attention, *prefill(start=2040, tokens=9), message=b"positions below 2048")
    refused(lib.pkv_fp8_prefill_attention, *prefill(bytes=2 * 16388 - 1), message=b"workspace")
    refused(lib.pkv_fp8_prefill_attention, *prefill(fp32=1, stride=2044), message=b"2048 or more")
    refused(lib.pkv_fp8_prefill_attention, *prefill(blocks=None), message=b"null pointer")
    refused(lib.pkv_fp8_prefill_attention, *prefill(layer=2), message=b"layers out of range")
    out, size = ctypes.c_int32(), ctypes.c_int64()
    refused(lib.pkv_fp8_decode_plan, 0, 0, 4, ctypes.byref(out), ctypes.byref(size), message=b"nonempty batch")


def test_tensors_on_the_cpu_are_refused() -> None:
    half = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize_rows(half)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.add_rms_norm(half, None, half[0])
    with pytest.raises(ValueError, match="CUDA"):
        fp8.Fp8Cache.empty(1, 1, "cpu")
    weight = fp8.quantize_weight(torch.randn(4, 64))  # made anywhere, used on the GPU
    with pytest.raises(ValueError, match="CUDA"):
        fp8.linear(fp8.Fp8Rows(torch.zeros(2, 64).to(torch.float8_e4m3fn), torch.ones(2, 1)), weight)


def test_rows_that_overlap_are_refused() -> None:
    row = torch.zeros(1, 64)
    assert fp8._row_stride("x", row, 64) == 64
    assert fp8._row_stride("x", row[:, :32], 32) in (32, 64)
    assert fp8._row_stride("x", torch.zeros(3, 80)[:, :64], 64) == 80
    for overlapping in (row.expand(3, 64), torch.zeros(128).as_strided((3, 64), (32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            fp8._row_stride("x", overlapping, 64)


@pytest.mark.parametrize("n, k", [(1, 16), (130, 128), (300, 400)])
def test_quantize_weight_is_one_rounding_with_the_block_scale(n, k) -> None:
    generator = torch.Generator().manual_seed(n)
    weight = torch.randn(n, k, generator=generator) * torch.exp2(torch.randn(n, 1, generator=generator) * 3)
    result = fp8.quantize_weight(weight)
    scales = torch.zeros(-(-n // 128), -(-k // 128), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            scales[i, j] = scale_for(weight[128 * i : 128 * i + 128, 128 * j : 128 * j + 128].abs().max())
    assert torch.equal(result.scales.double(), scales)
    each = scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    assert torch.equal(result.codes.double() * each, round_e4m3(weight.double(), each))


def test_quantize_weight_at_the_ends_of_the_range() -> None:
    weight = torch.zeros(2, 144)
    weight[0, :4] = torch.tensor([70000.0, -1.0, float("inf"), 3.0])
    weight[1, 130:133] = torch.tensor([float("nan"), 2.0**-30, 0.0])
    result = fp8.quantize_weight(weight)
    assert result.scales.tolist() == [[256.0, 2.0**-15]]
    values = result.codes.float() * torch.tensor([[256.0] * 128 + [2.0**-15] * 16])
    assert values[0, 0] == 61440 and values[0, 2].isnan() and values[1, 130].isnan()
    assert values[1, 131] == 0 and values[0, 3] == 3.0
