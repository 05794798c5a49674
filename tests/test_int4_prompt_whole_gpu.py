"""Prompt attention over the 4-bit cache, every token of a chunk, by rows, by tiles and by tiles in parts."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import int4
from tests.fp8_reference import HALF_FP16, attend64
from tests.int4_reference import LAYER, Case
from tests.test_int4_gpu import randn

pytestmark = pytest.mark.gpu

# By rows; by tiles; in parts, whose ends fall inside, on and behind the positions of a tile.
CHUNKS = [(0, 33), (49, 31), (601, 75), (0, 300), (63, 257), (319, 176), (325, 176), (383, 200), (450, 176), (1000, 512),
          (1039, 701), (1500, 220), (1500, 548), (1535, 300), (1777, 271)]


@pytest.mark.parametrize("start, tokens", CHUNKS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_token_of_a_chunk(start, tokens, dtype) -> None:
    case = Case(start + tokens, [start + tokens], spread=0.5)
    query = (2 * randn(1, tokens, 32, 64)).to(dtype)
    out = int4.prefill_attention(case.cache, LAYER, query, case.batch()[2], start, case.flag)
    assert int(case.flag.item()) == 0
    key, value = case.tokens(0)
    for t in range(tokens):
        exact, bound = attend64(query[t], key[: start + t + 1], value[: start + t + 1], HALF_FP16)
        assert bool(((out[t].double() - exact).abs() <= bound).all()), t
