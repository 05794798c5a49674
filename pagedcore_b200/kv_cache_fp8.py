"""The KV allocator over an 8-bit cache.

``Fp8KVAllocator`` is :class:`KVAllocator` (same bookkeeping, calls, errors and
transactions) whose storage is an :class:`pagedcore_b200.fp8.Fp8Cache`: half
the bytes per token, so twice the tokens in the same memory and half the
traffic of a decode step.  The decoder functions, the step graphs and the
scheduler take it in place of a ``KVAllocator``.

What differs: K and V are rounded to E4M3 with a scale per block of 16 tokens
and head (K rotated in FP32 and rounded once), a prompt chunk's rotated queries
are FP32 (``prompt_query_dtype``) unless rotated in place, ``read_block`` and
``iter_layer_blocks`` return FP16 copies of what is stored instead of views,
and a token that raises its block's scale may round the block's earlier codes
again.  A step or prompt chunk that fails leaves the cache as it was: the open
blocks are copied before it (8 KiB a row and layer) and put back.
"""

from __future__ import annotations

from collections.abc import Iterator

import torch
from torch import Tensor

from pagedcore_b200 import fp8
from pagedcore_b200._lib import check, lib
from pagedcore_b200.config import PagedCoreConfig
from pagedcore_b200.engine_types import RequestId
from pagedcore_b200.kv_cache import _BLOCK_TOKENS, _LAYERS, DecodeBatch, KVAllocator

_BLOCK_BYTES = _LAYERS * 2 * 4 * (_BLOCK_TOKENS * 64 + 4)  # codes and one FP32 scale per head


def allocate_fp8_kv_pool(config: PagedCoreConfig, *, device: str | torch.device = "cuda:0") -> fp8.Fp8Cache:
    """``allocate_kv_pool`` for an 8-bit cache: as many blocks as ``kv_pool_mib`` holds."""
    target = torch.device(device)
    if target.type != "cuda":
        raise ValueError("KV pool requires a CUDA device")
    if not torch.cuda.is_available():
        raise RuntimeError("KV pool requires an available CUDA runtime")
    pool_bytes = config.kv_pool_mib * 2**20
    margin_bytes = config.workspace_margin_mib * 2**20
    if torch.cuda.mem_get_info(target)[0] < pool_bytes + margin_bytes:
        raise RuntimeError("configured KV pool and workspace margin do not fit in GPU memory")
    cache = fp8.Fp8Cache.empty(_LAYERS, pool_bytes // _BLOCK_BYTES, target)
    if torch.cuda.mem_get_info(target)[0] < margin_bytes:
        del cache
        raise RuntimeError("KV pool allocation leaves less than the configured workspace margin")
    return cache


class Fp8KVAllocator(KVAllocator):
    """Assign blocks within an 8-bit cache of 22 layers."""

    prompt_query_dtype = torch.float32  # rotated in FP32 and not rounded

    def __init__(self, pool: fp8.Fp8Cache, *, validation: str = "full") -> None:
        if not isinstance(pool, fp8.Fp8Cache) or pool.layers != _LAYERS:
            raise ValueError("KV pool must be an 8-bit cache of 22 layers")
        self._setup(pool, pool.num_blocks, validation, "rows")

    # -- the cache's kernels ------------------------------------------------------
    def _write(
        self, key: Tensor, value: Tensor, slots: Tensor, layer_begin: int, *, positions: Tensor | None = None,
        query_in: Tensor | None = None, query_out: Tensor | None = None,
    ) -> None:
        fp8.append_kv(
            self._pool, key, value, slots, layer_begin=layer_begin, error_flag=self._error, positions=positions,
            rope_table=None if positions is None else self._rope, query=query_in, query_out=query_out,
        )

    def _attend_prompt(self, layer: int, query: Tensor, blocks: Tensor, start: int, out: Tensor) -> Tensor:
        return fp8.prefill_attention(self._pool, layer, query, blocks, start, self._error, out)

    def attend(self, batch: DecodeBatch, query: Tensor, *, layer_index: int, out: Tensor | None = None) -> Tensor:
        """Decode attention of FP16 query [B, 32, 64] over a :class:`DecodeBatch` (FP32 is rounded first)."""
        self._check_worker()
        if query.dtype == torch.float32:
            query = query.half()
        to = self._aligned_out(out)
        result = fp8.decode_attention(
            self._pool, layer_index, query, batch.lengths, batch.prefix, batch.flat, batch.total_blocks, self._error,
            to,
        )
        return result if to is out else out.copy_(result)

    @staticmethod
    def _aligned_out(out: Tensor | None) -> Tensor | None:
        """``out`` [rows, 32, 64], or rows to copy to it where its own are not what the kernels write."""
        if out is None:
            return None
        if out.ndim != 3 or out.dtype != torch.float16 or out.stride()[1:] != (64, 1):
            raise ValueError("out must be FP16 [batch, 32, 64] with contiguous rows")
        fp8._row_stride("out", out, 32 * 64)
        if fp8._rows_ok(out, out.stride()):
            return out
        return torch.empty_like(out, memory_format=torch.contiguous_format)

    def _decode_layer_args(self, batch: DecodeBatch, rows: int, grid: int) -> tuple:
        grid = fp8.decode_plan(self._pool.device.index, rows, batch.total_blocks)[0]
        return self._layer_args(batch, rows, grid, batch.total_blocks)

    def _replay_args(self, rows: int, grid: int) -> tuple:
        # The kernels read the batch's block count on the device; the grid is every resident slot.
        capacity = self._staged.flat_capacity
        grid = fp8.decode_plan(self._pool.device.index, rows, 1 << 24)[0]
        return self._layer_args(self._staged.staged_batch, rows, grid, capacity)

    def _layer_args(self, batch: DecodeBatch, rows: int, grid: int, capacity: int) -> tuple:
        workspace = self._workspace_for(fp8.decode_workspace_bytes(rows, grid))
        return (
            self._pool._args(), self._rope.data_ptr(), batch.lengths.data_ptr(), batch.prefix.data_ptr(),
            batch.flat.data_ptr(), capacity, grid, workspace.data_ptr(), workspace.numel() * 4, self._error.data_ptr(),
        )

    def _launch_decode_layer(
        self, layer: int, query: Tensor, key: Tensor, value: Tensor, out: Tensor, rows: int, fixed: tuple,
        flags: int, stream: int,
    ) -> None:
        cache, rope, lengths, prefix, flat, capacity, grid, workspace, workspace_bytes, error = fixed
        query, query_stride = fp8._query_rows(query)
        key, value, strides = fp8._aligned_pair(key, value)
        to = self._aligned_out(out)
        if to is not out:
            to.copy_(out)  # rows past the batch are left alone
        check(
            lib.pkv_fp8_decode_layer(
                *cache, layer, query.data_ptr(), query_stride, key.data_ptr(), value.data_ptr(), strides[0], rope,
                lengths, prefix, flat, rows, capacity, grid, to.data_ptr(), fp8._row_stride("out", to, 32 * 64),
                workspace, workspace_bytes, error, stream,
            )
        )
        if to is not out:
            out.copy_(to)

    def _save_blocks(self, slots: Tensor) -> tuple[Tensor, Tensor]:
        return slots, fp8.save_blocks(self._pool, slots)

    def _restore_blocks(self, saved: tuple[Tensor, Tensor]) -> None:
        fp8.restore_blocks(self._pool, *saved)

    # -- reading back ----------------------------------------------------------------
    @torch.inference_mode()
    def iter_layer_blocks(self, request_id: RequestId, *, layer_index: int) -> Iterator[tuple[Tensor, Tensor]]:
        """FP16 copies of the valid [slots, 4, 64] pages, including a completed staged layer."""
        self._check_worker()
        if type(layer_index) is not int or not 0 <= layer_index < _LAYERS:
            raise ValueError("layer_index must identify one of the 22 decoder layers")
        blocks, length = self._call(self._ledger.view, request_id, self._handle(request_id), layer_index)
        if length == 0:
            raise ValueError("attention requires a nonempty cache")
        for logical, physical in enumerate(blocks):
            self._check_worker()
            valid = min(_BLOCK_TOKENS, length - logical * _BLOCK_TOKENS)
            key, value = self._read(layer_index, physical)
            yield key[:valid], value[:valid]

    @torch.inference_mode()
    def read_block(self, request_id: RequestId, logical_block: int) -> tuple[Tensor, Tensor]:
        """FP16 copies of K/V [22, valid slots, 4, 64] of one logical block."""
        self._check_worker()
        handle = self._handle(request_id)
        blocks = self._call(self._ledger.table, request_id, handle)
        length = self._ledger.length(handle)
        if type(logical_block) is not int or not 0 <= logical_block < len(blocks):
            raise ValueError("logical block must identify a cached block")
        valid = min(_BLOCK_TOKENS, length - logical_block * _BLOCK_TOKENS)
        layers = [self._read(layer, blocks[logical_block]) for layer in range(_LAYERS)]
        return tuple(torch.stack([layer[kv][:valid] for layer in layers]) for kv in (0, 1))

    def _read(self, layer: int, physical: int) -> tuple[Tensor, Tensor]:
        block = torch.full((1,), physical, dtype=torch.int32, device=self._pool.device)
        key, value = fp8.read_blocks(self._pool, layer, block, self._error)
        return key[0], value[0]
