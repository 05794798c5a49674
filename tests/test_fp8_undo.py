"""A failed step or prompt chunk leaves an 8-bit cache as it was, codes and scales."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import _lib, fp8
from pagedcore_b200.graph import DecodeStepGraph
from tests.test_fp8_capi import CACHE, P, lib, refused


def test_refusals() -> None:
    size = 2 * 3 * 8224
    refused(lib.pkv_fp8_save_blocks, P, None, P, P, 2, 8, P, 3, P, size, 0, None, message=b"codes and scales")
    refused(lib.pkv_fp8_save_blocks, *CACHE, None, 3, P, size, 0, None, message=b"slots")
    refused(lib.pkv_fp8_save_blocks, *CACHE, P, -1, P, size, 0, None, message=b"slots")
    refused(lib.pkv_fp8_save_blocks, *CACHE, P, 3, None, size, 1, None, message=b"buffer")
    refused(lib.pkv_fp8_save_blocks, *CACHE, P, 3, P, size - 1, 0, None, message=b"8224 bytes")
    refused(lib.pkv_fp8_save_blocks, *CACHE, P, 3, P + 8, size, 1, None, message=b"16-byte")
    assert lib.pkv_fp8_save_blocks(*CACHE, P, 0, P, 0, 0, None) == _lib.PKV_OK


def filled(lengths):
    from tests.test_fp8_decoder_gpu import admit, make_allocator
    from tests.test_fp8_gpu import randn

    allocator = make_allocator(sum(-(-n // 16) + 4 for n in lengths))
    requests = admit(allocator, *[-(-n // 16) + 4 for n in lengths])
    for i, (request, n) in enumerate(zip(requests, lengths)):
        allocator.append(request, randn(500 + i, 22, n, 4, 64).half(), randn(510 + i, 22, n, 4, 64).half(), rotate=True)
    return allocator, requests


def snapshot(allocator, requests):
    """Codes of the valid slots, and scales, of every request in every layer."""
    cache, state = allocator.pool, []
    for request in requests:
        length = allocator.cached_length(request)
        for logical, block in enumerate(allocator.block_table(request)):
            valid = min(16, length - 16 * logical)
            state += [cache.key_codes.view(torch.uint8)[:, block, :, :valid].clone(),
                      cache.value_codes.view(torch.uint8)[:, block, :, :, :valid].clone(),
                      cache.key_scales[:, block].clone(), cache.value_scales[:, block].clone()]
    return state


def same(a, b) -> bool:
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def tokens(seed: int, count: int, factor: float):
    """Queries, keys and values of `count` tokens of magnitudes that raise every scale."""
    from tests.test_fp8_gpu import randn

    return [(factor * randn(seed + heads, count, heads, 64)).half() for heads in (32, 4, 4)]


LENGTHS = [20, 16, 1, 47, 31]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["layer", "batch", "row", "commit"])
def test_a_failed_decode_step_leaves_the_cache_as_it_was(how) -> None:
    allocator, requests = filled(LENGTHS)
    twin, twins = filled(LENGTHS)
    before = snapshot(allocator, requests)
    q, k, v = tokens(520, len(LENGTHS), 300.0)
    with pytest.raises(RuntimeError, match="every cache layer" if how == "commit" else "boom"):
        with allocator.append_decode(requests):
            for layer in range(21 if how == "commit" else 22):
                if how == "batch":
                    allocator.write_decode_batch(layer, k, v, query=q, rotate=True)
                elif how == "row":
                    for row, request in enumerate(requests):
                        allocator.write_decode_layer(request, layer, k[row], v[row])
                else:
                    allocator.decode_layer(layer, q, k, v)
            assert not same(snapshot(allocator, requests), before)  # the step did round earlier codes again
            if how != "commit":
                raise RuntimeError("boom")
    assert same(snapshot(allocator, requests), before)
    # The next step is that of a cache in which nothing failed.
    q, k, v = tokens(530, len(LENGTHS), 1.0)
    for side, ids in ((allocator, requests), (twin, twins)):
        with side.append_decode(ids):
            outs = [side.decode_layer(layer, q, k, v) for layer in range(22)]
        side.check_device_errors()
        if side is allocator:
            expected = outs
    assert same(outs, expected) and same(snapshot(allocator, requests), snapshot(twin, twins))


@pytest.mark.gpu
def test_a_step_graph_that_fails_behind_its_replay_leaves_the_cache_as_it_was(monkeypatch) -> None:
    allocator, requests = filled(LENGTHS)
    rows = len(LENGTHS) + 1
    from tests.test_fp8_gpu import randn

    q, k, v = (randn(540 + heads, 22, rows, heads, 64).half() for heads in (32, 4, 4))
    out = torch.zeros(22, rows, 32, 64, dtype=torch.float16, device=q.device)
    graph = DecodeStepGraph(allocator, rows=rows)
    graph.step(q, k, v, out, requests)
    before = snapshot(allocator, requests)
    k.mul_(200)
    v.mul_(200)

    def commit():
        assert not same(snapshot(allocator, requests), before)
        raise RuntimeError("boom")

    with monkeypatch.context() as patch:
        patch.setattr(allocator.ledger, "decode_commit", commit)
        with pytest.raises(RuntimeError, match="boom"):
            graph.step(q, k, v, out, requests)
    allocator.ledger.decode_abort()
    assert same(snapshot(allocator, requests), before)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [20, 16, 31])
def test_a_failed_prompt_chunk_leaves_the_cache_as_it_was(length) -> None:
    allocator, (request,) = filled([length])
    before = snapshot(allocator, (request,))
    q, k, v = tokens(550, 40, 300.0)
    with pytest.raises(RuntimeError, match="boom"):
        with allocator.prefill_append(request, 40) as chunk:
            for layer in range(22):
                chunk.attend(layer, chunk.write_layer(layer, k, v, q))
            assert same(snapshot(allocator, (request,)), before) == (length == 16)
            raise RuntimeError("boom")
    assert same(snapshot(allocator, (request,)), before)


@pytest.mark.gpu
def test_a_failed_chunk_does_not_undo_what_others_wrote_meanwhile() -> None:
    from tests.test_fp8_gpu import randn

    allocator, (request,) = filled([20])
    with pytest.raises(RuntimeError, match="boom"):
        with allocator.prefill_append(request, 4):
            allocator.append(request, randn(560, 22, 3, 4, 64).half() * 50, randn(561, 22, 3, 4, 64).half() * 50)
            grown = snapshot(allocator, (request,))
            raise RuntimeError("boom")
    assert allocator.cached_length(request) == 23 and same(snapshot(allocator, (request,)), grown)


@pytest.mark.gpu
def test_save_and_restore_blocks() -> None:
    from tests.test_fp8_gpu import LAYERS, CacheCase

    case = CacheCase(561, [20, 16, 40])
    cache = case.cache
    names = ("key_codes", "value_codes", "key_scales", "value_scales")
    slots = torch.tensor([16 * case.tables[0][1] + 4, 16 * case.tables[1][0],
                          16 * case.tables[2][2] + 1, -1, 16 * cache.num_blocks + 3], dtype=torch.int32, device=case.device)
    before = [getattr(cache, name).view(torch.uint8).clone() for name in names]
    saved = fp8.save_blocks(cache, slots)
    assert saved.numel() == 5 * LAYERS * 8224
    assert all(torch.equal(a, getattr(cache, n).view(torch.uint8)) for a, n in zip(before, names))
    for name in names:
        getattr(cache, name).view(torch.uint8).fill_(0x11)
    fp8.restore_blocks(cache, slots, saved)
    touched = {case.tables[0][1], case.tables[2][2]}  # the others open their block, or lie outside the cache
    for old, name in zip(before, names):
        now = getattr(cache, name).view(torch.uint8)
        for block in range(cache.num_blocks):
            assert torch.equal(now[:, block], old[:, block]) if block in touched else bool((now[:, block] == 0x11).all())
    with pytest.raises(ValueError, match="saved"):
        fp8.restore_blocks(cache, slots, saved.view(torch.int8))
    with pytest.raises(ValueError, match="8224 bytes"):
        fp8.restore_blocks(cache, slots, saved[:8224])
