"""The KV allocator over a 4-bit cache.

``Int4KVAllocator`` is :class:`KVAllocator` (same bookkeeping, calls, errors and
transactions) whose storage is an :class:`pagedcore_b200.int4.Int4Cache`: 288 bytes
a token and layer where the FP16 pool has 1024, so 3.56 times the tokens in the
same memory (1.78 times the 8-bit cache's).  The decoder functions, the step graphs and the scheduler take it in
place of a ``KVAllocator``.

What differs: K and V are rounded to 4 bits with a scale per 16 dims (K rotated in
FP32 and rounded once), a prompt chunk's rotated queries are FP32
(``prompt_query_dtype``) unless rotated in place, and ``read_block`` and
``iter_layer_blocks`` return FP16 copies of what is stored instead of views.  No write
touches another token, so a step or prompt chunk that fails has nothing to put back.

With ``norms`` (the weights of a model's query and key norms), wherever K and the
queries are rotated here they are normed first; rows that come rotated
(``append`` and ``write_decode_batch`` without ``rotate``, ``write_decode_layer``) are
written as they are.
"""

from __future__ import annotations

import torch
from torch import Tensor

from pagedcore_b200 import fp8, int4
from pagedcore_b200._lib import check, lib
from pagedcore_b200.config import PagedCoreConfig
from pagedcore_b200.kv_cache import _LAYERS, DecodeBatch
from pagedcore_b200.kv_cache_quantised import QuantisedKVAllocator, allocate_quantised


def allocate_int4_kv_pool(config: PagedCoreConfig, *, device: str | torch.device = "cuda:0") -> int4.Int4Cache:
    """``allocate_kv_pool`` for a 4-bit cache: as many blocks as ``kv_pool_mib`` holds."""
    return allocate_quantised(
        config, device, _LAYERS * int4.BLOCK_BYTES, lambda blocks, on: int4.Int4Cache.empty(_LAYERS, blocks, on)
    )


class Int4KVAllocator(QuantisedKVAllocator):
    """Assign blocks within a 4-bit cache of 22 layers."""

    def __init__(
        self, pool: int4.Int4Cache, *, validation: str = "full", norms: int4.HeadNorms | None = None
    ) -> None:
        if not isinstance(pool, int4.Int4Cache) or pool.layers != _LAYERS:
            raise ValueError("KV pool must be a 4-bit cache of 22 layers")
        if norms is not None:
            norms.check(pool)
        self._norms = norms
        self._setup(pool, pool.num_blocks, validation, "rows")

    # -- the cache's kernels ------------------------------------------------------
    def _write(
        self, key: Tensor, value: Tensor, slots: Tensor, layer_begin: int, *, positions: Tensor | None = None,
        query_in: Tensor | None = None, query_out: Tensor | None = None,
    ) -> None:
        rotate = positions is not None
        int4.append_kv(
            self._pool, key, value, slots, layer_begin=layer_begin, error_flag=self._error, positions=positions,
            rope_table=self._rope if rotate else None, query=query_in, query_out=query_out,
            norms=self._norms if rotate else None,
        )

    def _attend_prompt(self, layer: int, query: Tensor, blocks: Tensor, start: int, out: Tensor) -> Tensor:
        return int4.prefill_attention(self._pool, layer, query, blocks, start, self._error, out)

    def _attend_rows(self, layer: int, batch: DecodeBatch, query: Tensor, out: Tensor | None) -> Tensor:
        return int4.decode_attention(
            self._pool, layer, query, batch.lengths, batch.prefix, batch.flat, batch.total_blocks, self._error, out
        )

    def _decode_layer_args(self, batch: DecodeBatch, rows: int, grid: int) -> tuple:
        grid = int4.decode_plan(self._pool.device.index, rows, batch.total_blocks)[0]
        return self._layer_args(batch, rows, grid, batch.total_blocks)

    def _replay_args(self, rows: int, grid: int) -> tuple:
        # The kernels read the batch's block count on the device; the grid is every resident slot.
        capacity = self._staged.flat_capacity
        grid = int4.decode_plan(self._pool.device.index, rows, 1 << 24)[0]
        return self._layer_args(self._staged.staged_batch, rows, grid, capacity)

    def _layer_args(self, batch: DecodeBatch, rows: int, grid: int, capacity: int) -> tuple:
        workspace = self._workspace_for(int4.decode_workspace_bytes(rows, grid))
        norms = self._norms
        return (
            self._pool._args(), self._rope.data_ptr(),
            (None, None, 0.0) if norms is None else (norms.query.data_ptr(), norms.key.data_ptr(), norms.eps),
            batch.lengths.data_ptr(), batch.prefix.data_ptr(), batch.flat.data_ptr(), capacity, grid,
            None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel() * 4,
            self._error.data_ptr(),
        )

    def _launch_decode_layer(
        self, layer: int, query: Tensor, key: Tensor, value: Tensor, out: Tensor, rows: int, fixed: tuple,
        flags: int, stream: int,
    ) -> None:
        cache, rope, norms, lengths, prefix, flat, capacity, grid, workspace, workspace_bytes, error = fixed
        query, query_stride = fp8._query_rows(query)
        key, value, strides = fp8._aligned_pair(key, value)
        to = self._aligned_out(out)
        if to is not out:
            to.copy_(out)  # rows past the batch are left alone
        elif int4.overlaps(query, out):
            query, query_stride = fp8._dense(query), 32 * 64
        if int4.overlaps(key, to) or int4.overlaps(value, to):
            key, value = fp8._dense(key), fp8._dense(value)
            strides = key.stride()
        check(
            lib.pkv_int4_decode_layer(
                *cache, layer, query.data_ptr(), query_stride, key.data_ptr(), value.data_ptr(), strides[0], rope, *norms,
                lengths, prefix, flat, rows, capacity, grid, 0, to.data_ptr(), fp8._row_stride("out", to, 32 * 64),
                workspace, workspace_bytes, error, stream,
            )
        )
        if to is not out:
            out.copy_(to)

    # -- reading back ----------------------------------------------------------------
    def _read(self, layer: int, physical: int) -> tuple[Tensor, Tensor]:
        block = torch.full((1,), physical, dtype=torch.int32, device=self._pool.device)
        key, value = int4.read_blocks(self._pool, layer, block, self._error)
        return key[0], value[0]
