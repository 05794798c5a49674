"""What the KV allocators over quantised caches share.

Their storage holds K and V rounded to fewer bits, so blocks are read back as
FP16 copies instead of views, a prompt chunk's rotated queries stay FP32, and
outputs that the kernels cannot write go through rows that they can.
"""

from __future__ import annotations

from collections.abc import Callable, Iterator

import torch
from torch import Tensor

from pagedcore_b200 import fp8
from pagedcore_b200.config import PagedCoreConfig
from pagedcore_b200.engine_types import RequestId
from pagedcore_b200.kv_cache import _BLOCK_TOKENS, _LAYERS, DecodeBatch, KVAllocator


def allocate_quantised(
    config: PagedCoreConfig, device: str | torch.device, block_bytes: int, make: Callable[[int, torch.device], object]
):
    """``make(blocks, device)`` with as many blocks of ``block_bytes`` as ``kv_pool_mib`` holds (``allocate_kv_pool``'s checks)."""
    target = torch.device(device)
    if target.type != "cuda":
        raise ValueError("KV pool requires a CUDA device")
    if not torch.cuda.is_available():
        raise RuntimeError("KV pool requires an available CUDA runtime")
    pool_bytes = config.kv_pool_mib * 2**20
    margin_bytes = config.workspace_margin_mib * 2**20
    if torch.cuda.mem_get_info(target)[0] < pool_bytes + margin_bytes:
        raise RuntimeError("configured KV pool and workspace margin do not fit in GPU memory")
    cache = make(pool_bytes // block_bytes, target)
    if torch.cuda.mem_get_info(target)[0] < margin_bytes:
        del cache
        raise RuntimeError("KV pool allocation leaves less than the configured workspace margin")
    return cache


class QuantisedKVAllocator(KVAllocator):
    """``KVAllocator`` over a cache object that has ``device`` and ``num_blocks``."""

    prompt_query_dtype = torch.float32  # rotated in FP32 and not rounded

    # -- the cache's kernels ------------------------------------------------------
    def _attend_rows(self, layer: int, batch: DecodeBatch, query: Tensor, out: Tensor | None) -> Tensor:
        """Decode attention of FP16 ``query`` at ``layer`` into ``out`` (rows that the kernels write, or None)."""
        raise NotImplementedError

    def _read(self, layer: int, physical: int) -> tuple[Tensor, Tensor]:
        """FP16 K and V [16, 4, 64] of one block."""
        raise NotImplementedError

    def attend(self, batch: DecodeBatch, query: Tensor, *, layer_index: int, out: Tensor | None = None) -> Tensor:
        """Decode attention of FP16 query [B, 32, 64] over a :class:`DecodeBatch` (FP32 is rounded first)."""
        self._check_worker()
        if query.dtype == torch.float32:
            query = query.half()
        to = self._aligned_out(out)
        result = self._attend_rows(layer_index, batch, query, to)
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
