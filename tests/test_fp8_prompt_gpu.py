"""Prompt attention over the 8-bit cache: nothing but the output is rounded to FP16."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8
from tests.fp8_reference import attend64
from tests.test_fp8_gpu import LAYER, CacheCase, randn

pytestmark = pytest.mark.gpu


def check_prompt(out, query, key, value, start: int, tokens) -> None:
    """Rows ``tokens`` of a chunk at ``start`` against 64 bits over K/V [tokens, 4, 64].

    ``attend64`` with the weights as the decode kernels have them, 2^-21: an
    FP16 number and what it leaves as another.  The smallest FP16 step adds
    2^-25 a weight where the largest one is 2^7 or more: 2^-32 of the largest V.
    """
    for t in tokens:
        k, v = key[: start + t + 1], value[: start + t + 1]
        exact, bound = attend64(query[t], k, v)
        bound = bound + len(k) * 2.0**-32 * v.abs().amax()
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t


@pytest.mark.parametrize("start, tokens", [(0, 1), (0, 15), (0, 130), (7, 40), (100, 64), (601, 75), (0, 2047), (2000, 48)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_attention_does_not_round_its_weights(start, tokens, dtype) -> None:
    case = CacheCase(131, [start + tokens])
    query = randn(132, tokens, 32, 64).to(dtype)
    out = fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert int(case.flag.item()) == 0
    key, value = (oracle.tokens(case.tables[0], start + tokens) for oracle in (case.key, case.value))
    check_prompt(out, query, key, value, start, sorted({0, 1, 14, tokens // 3, tokens // 2, tokens - 1} & set(range(tokens))))
    assert torch.equal(fp8.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag), out)
