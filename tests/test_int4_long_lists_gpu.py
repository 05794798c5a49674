"""A row whose block list goes on past 2^31 tokens, of which only the first ones are its own."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import int4
from tests.int4_reference import LAYER, Case
from tests.test_int4_gpu import check_rows, randn

pytestmark = pytest.mark.gpu


def test_blocks_behind_a_rows_length_do_not_count_however_many_they_are() -> None:
    case = Case(71, [40, 20])
    spare = 2**27 + 64
    own, other = case.tables
    flat = torch.full((len(own) + spare + len(other),), case.free[0], dtype=torch.int32, device=case.device)  # a block of NaN
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=case.device)  # noqa: E731
    flat[: len(own)], flat[-len(other) :] = as_int(own), as_int(other)
    query = randn(72, 2, 32, 64).half()
    prefix = as_int([0, len(own) + spare, flat.numel()])
    out = int4.decode_attention(case.cache, LAYER, query, as_int(case.lengths), prefix, flat, flat.numel(), case.flag)
    assert int(case.flag.item()) == 0
    check_rows(case, query.double(), out)
