"""Sizes past the 32 bits of the 4-bit operators' C entry points are refused, on the host."""

from __future__ import annotations

import ctypes

import pytest

from tests.test_int4_capi import CACHE, P, lib, refused

MOST = 2**31 - 1


@pytest.mark.parametrize("tokens", [MOST, MOST - 2, MOST - 60000])
def test_append_refuses_tokens_whose_index_would_wrap(tokens) -> None:
    refused(lib.pkv_int4_append_kv, *CACHE, 0, 1, P, P, 0, 256, P, None, tokens, None, None, None, 1e-5, None, 0, 0, None,
            0, 0, 0, P, None, message=b"too many tokens")


@pytest.mark.parametrize("batch, total", [(1, MOST), (1, MOST - 60), (MOST, 4), (MOST - 10_000_000, 4)])
def test_decode_refuses_lists_and_batches_whose_loops_would_wrap(batch, total) -> None:
    tables = (P, P, P, batch, total, 4)
    rest = (P, 2048, P, 2**60, P, None)
    refused(lib.pkv_int4_decode_attention, *CACHE, 0, P, 2048, *tables, *rest, message=b"out of range")
    refused(lib.pkv_int4_decode_layer, *CACHE, 0, P, 2048, P, P, 256, P, None, None, 1e-5, *tables, 1, *rest, message=b"out of range")
    refused(lib.pkv_int4_decode_plan, 0, batch, total, ctypes.byref(ctypes.c_int32()), ctypes.byref(ctypes.c_int64()),
            message=b"out of range")
