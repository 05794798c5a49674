"""What an allocator over the 4-bit cache checks once cannot be replaced behind it."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from pagedcore_b200 import int4
from tests.conftest import cuda_device


def test_head_norms_keep_their_weights() -> None:
    weight = torch.ones(22, 64, dtype=torch.float16)
    norms = int4.HeadNorms(weight, weight)
    for name, other in (("query", weight[:1]), ("key", weight.float()), ("eps", -1.0)):
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(norms, name, other)
    assert norms.query is weight and norms.key is weight and norms.eps == 1e-5


@pytest.mark.gpu
def test_a_cache_keeps_its_storage() -> None:
    cache = int4.Int4Cache.empty(2, 3, cuda_device())
    with pytest.raises(dataclasses.FrozenInstanceError):
        cache.storage = cache.storage[:, :1]
    assert cache.num_blocks == 3
