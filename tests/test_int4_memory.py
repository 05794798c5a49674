"""The memory figures that the 4-bit cache's documentation gives."""

from __future__ import annotations

from pagedcore_b200 import int4, kv_cache, kv_cache_fp8, kv_cache_int4


def test_bytes_of_a_token_in_each_cache() -> None:
    tokens = kv_cache._BLOCK_TOKENS
    four = int4.BLOCK_BYTES // tokens
    half = 2 * 4 * 64 * 2  # K and V of 4 heads of 64 dims in FP16
    eight = kv_cache_fp8._BLOCK_BYTES // (kv_cache._LAYERS * tokens)
    assert f"{four} bytes a layer, FP16 {half} and E4M3 {eight}" in int4.__doc__
    text = " ".join(kv_cache_int4.__doc__.split())
    assert f"{four} bytes a token and layer where the FP16 pool has {half}, so {half / four:.2f} times the tokens" in text
    assert f"{eight / four:.2f} times the 8-bit cache's" in text
