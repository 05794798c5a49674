"""Sizes past the 32 bits of the 8-bit operators' C entry points are refused, on the host."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8
from tests.test_fp8_capi import P, lib, refused

MOST = 2**31 - 1


def test_the_entry_points_refuse_sizes_whose_loops_would_wrap() -> None:
    refused(lib.pkv_fp8_add_rms_norm, P, None, P, None, P, P, MOST, 64, 1e-5, None, message=b"too many rows")
    refused(lib.pkv_fp8_quantize, P, 64, 0, MOST - 100, 64, P, P, None, message=b"too many rows")
    refused(lib.pkv_fp8_to_half, P, P, MOST - 65534, 16, P, 16, None, message=b"too many rows")
    for rows, n, k in ((MOST, 8, 64), (MOST - 100, 8, 64), (8, MOST, 64), (8, 8, MOST // 16 * 16)):
        refused(lib.pkv_fp8_linear, P, k, P, P, P, rows, n, k, P, n, P, None, message=b"too many rows or columns")


@pytest.mark.parametrize("rows", [2**31, 2**32 + 5])
def test_tensors_past_32_bits_are_refused(rows) -> None:
    meta = lambda *shape, dtype=torch.float16: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="rows must be at most"):
        fp8.quantize_rows(meta(rows, 8))
    with pytest.raises(ValueError, match="rows must be at most"):
        fp8.silu_mul(meta(rows, 16))
    with pytest.raises(ValueError, match="rows must be at most"):
        fp8.add_rms_norm(meta(rows, 8), None, meta(8))
    many = fp8.Fp8Rows(meta(rows, 16, dtype=torch.float8_e4m3fn), meta(rows, 1, dtype=torch.float32))
    few = fp8.Fp8Rows(meta(3, 16, dtype=torch.float8_e4m3fn), meta(3, 1, dtype=torch.float32))
    with pytest.raises(ValueError, match="rows must be at most"):
        many.to_half()
    with pytest.raises(ValueError, match="rows must be at most"):
        fp8.linear(many, fp8.Fp8Weight(few.codes, few.scales[:1]))
    with pytest.raises(ValueError, match="n must be at most"):
        fp8.linear(few, fp8.Fp8Weight(many.codes, meta(-(-rows // 128), 1, dtype=torch.float32)))
    with pytest.raises(ValueError, match="entries of slots must be at most"):
        fp8._int_list(0, "slots", torch.zeros(4, dtype=torch.int32), rows)
