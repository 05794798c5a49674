"""The KV cache in 4 bits, and the operators over it.

The 4-bit forms of the FP16 operators in :mod:`pagedcore_b200.kernels` and of the
8-bit ones in :mod:`pagedcore_b200.fp8`, in the same manner (tensor checks here,
work in the sm_100a kernels, the current CUDA stream of the tensors' device):
``append_kv`` writes K and V into an :class:`Int4Cache`, ``read_blocks`` reads them
back, ``decode_layer``, ``decode_attention`` and ``prefill_attention`` attend to them.

A group is 16 consecutive dims of one token and head: 16 codes from -7 to 7 and
one scale of 8 bits (5 exponent and 3 fraction bits, no sign), a value being code
times scale, an FP16 number.  A written value moves by at most half its group's
scale, which is about a seventh of the group's largest magnitude (values past
64512 are held as that); a group with a value that is not finite reads as NaN.
A token takes 288 bytes a layer, FP16 2048 and E4M3 1026.

With :class:`HeadNorms`, queries and keys are normed head by head before they
are rotated, in the same pass.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch
from torch import Tensor

from pagedcore_b200._lib import check, lib
from pagedcore_b200.fp8 import (
    _ROW,
    _aligned_pair,
    _attention_rows,
    _call,
    _check_rope,
    _dense,
    _fits,
    _half,
    _int_list,
    _mixes,
    _query_and_out,
    _rows_apart,
    _rows_ok,
)

BLOCK_BYTES = 4608  # of 16 tokens in one layer
_KV_HEADS = 4
_QUERY_HEADS = 32
_HEAD_DIM = 64
_BLOCK_TOKENS = 16
_BYTE = torch.uint8
_HALF = torch.float16
_FLOAT = torch.float32


@dataclass(slots=True)
class Int4Cache:
    """A 4-bit KV cache: bytes [layers, blocks, 4608].

    A block holds 16 tokens: for each of the 4 heads 512 bytes of K codes [4 groups,
    16 tokens, 8], 512 of V codes [8 chunks of 8 dims, 16 tokens, 4], 64 of K scales
    [4 groups, 16 tokens] and 64 of V scales (``include/pagedkv.h`` gives the order of
    the codes).  A slot id is physical_block * 16 + slot_in_block, as in the FP16 pool.
    """

    storage: Tensor

    def __post_init__(self) -> None:
        storage = self.storage
        shape = storage.shape
        if len(shape) != 3 or shape[2] != BLOCK_BYTES or storage.dtype is not _BYTE or not storage.is_contiguous():
            raise ValueError("a 4-bit cache is contiguous uint8 [layers, blocks, 4608]")
        if shape[0] < 1 or shape[1] < 1:
            raise ValueError("a 4-bit cache needs at least one layer and one block")
        if storage.get_device() < 0:
            raise ValueError("4-bit operators need CUDA tensors")

    @classmethod
    def empty(cls, layers: int, blocks: int, device: str | torch.device = "cuda") -> Int4Cache:
        """Uninitialised storage: only written, valid slots may be read."""
        return cls(torch.empty((layers, blocks, BLOCK_BYTES), dtype=_BYTE, device=device))

    @property
    def device(self) -> torch.device:
        return self.storage.device

    @property
    def layers(self) -> int:
        return self.storage.shape[0]

    @property
    def num_blocks(self) -> int:
        return self.storage.shape[1]

    def _args(self) -> tuple[int, int, int]:
        storage = self.storage
        shape = storage.shape
        return storage.data_ptr(), shape[0], shape[1]


@dataclass(slots=True)
class HeadNorms:
    """Weights of the RMS norms of each query and key head, FP16 [layers, 64] each, for a cache's layers.

    x * rsqrt(mean(x^2) + eps) * weight over the 64 dims of a head, before the rotation.
    """

    query: Tensor
    key: Tensor
    eps: float = 1e-5

    def _args(self, cache: Int4Cache) -> tuple[int, int, float]:
        query, key, eps = self.query, self.key, self.eps
        index, shape = cache.storage.get_device(), (cache.storage.shape[0], _HEAD_DIM)
        for tensor in (query, key):
            if (
                tensor.shape != shape
                or tensor.dtype is not _HALF
                or not tensor.is_contiguous()
                or tensor.get_device() != index
                or tensor.data_ptr() % 16
            ):
                raise ValueError(f"head norms must be contiguous, 16-byte aligned FP16 {list(shape)} on cuda:{index}")
        if not eps >= 0:
            raise ValueError("eps must not be negative")
        return query.data_ptr(), key.data_ptr(), eps


_NO_NORMS = (None, None, 0.0)


def append_kv(
    cache: Int4Cache,
    key: Tensor,
    value: Tensor,
    slots: Tensor,
    *,
    layer_begin: int,
    error_flag: Tensor,
    positions: Tensor | None = None,
    rope_table: Tensor | None = None,
    query: Tensor | None = None,
    query_out: Tensor | None = None,
    norms: HeadNorms | None = None,
) -> Tensor | None:
    """Write FP16 K/V [layers, tokens, 4, 64] into the cache at ``slots`` (int32 [tokens]).

    With ``rope_table`` K is rotated at ``positions`` first, and ``query``
    [layers, tokens, 32, 64] is returned rotated: in FP32, unrounded, for
    ``prefill_attention``, or in ``query_out``, FP16 (which may be ``query``
    itself) or FP32.  With ``norms`` each head of both is normed before it is
    rotated.  Tokens may go to any slots, in any order, but to no slot twice.
    """
    index = cache.storage.get_device()
    shape = key.shape
    if len(shape) != 4 or shape[2] != _KV_HEADS or shape[3] != _HEAD_DIM or value.shape != shape:
        raise ValueError("K and V must share FP16 [layers, tokens, 4, 64]")
    _half("key", key, index)
    _half("value", value, index)
    layers, tokens = shape[0], shape[1]
    _fits("layers", layers)
    slots_ptr = _int_list(index, "slots", slots, tokens)
    flag = _int_list(index, "error_flag", error_flag, 1)
    if (rope_table is None) != (positions is None) or (query is not None and rope_table is None):
        raise ValueError("rope_table goes with positions, query with both")
    rope = positions_ptr = None
    if rope_table is not None:
        rope = _check_rope(index, rope_table)
        positions_ptr = _int_list(index, "positions", positions, tokens)
    weights = _NO_NORMS
    if norms is not None:
        if rope is None:
            raise ValueError("norms go with rope_table")
        weights = norms._args(cache)
    q_ptr = out_ptr = None
    q_strides = out_strides = (0, 0)
    if query is not None:
        if query.shape != (layers, tokens, _QUERY_HEADS, _HEAD_DIM):
            raise ValueError("query must be FP16 [layers, tokens, 32, 64]")
        _half("query", query, index)
        given = query_out is not None
        if not given:
            query_out = torch.empty_like(query, dtype=_FLOAT, memory_format=torch.contiguous_format)
        elif (
            query_out.shape != query.shape
            or not _rows_ok(query_out, query_out.stride())
            or not _rows_apart(query_out.stride(), layers, tokens)
        ):
            raise ValueError("query_out must be [layers, tokens, 32, 64] with contiguous, 16-byte aligned rows")
        elif query_out.dtype not in (_HALF, _FLOAT) or query_out.get_device() != index:
            raise ValueError(f"query_out must be FP16 or FP32 on cuda:{index}")
        if not _rows_ok(query, query.stride()) or (given and _mixes(query, query_out)):
            query = _dense(query)
        q_ptr, out_ptr = query.data_ptr(), query_out.data_ptr()
        q_strides, out_strides = query.stride()[:2], query_out.stride()[:2]
    elif query_out is not None:
        raise ValueError("query_out goes with query")
    if layers == 0 or tokens == 0:
        return query_out
    key, value, strides = _aligned_pair(key, value)
    _call(index, lib.pkv_int4_append_kv, *cache._args(), layer_begin, layers, key.data_ptr(), value.data_ptr(),
          strides[0], strides[1], slots_ptr, positions_ptr, tokens, rope, *weights, q_ptr, *q_strides, out_ptr,
          query_out is not None and query_out.dtype is _FLOAT, *out_strides, flag)
    return query_out


def read_blocks(cache: Int4Cache, layer: int, blocks: Tensor, error_flag: Tensor) -> tuple[Tensor, Tensor]:
    """K and V of ``blocks`` (int32 [count]) at ``layer`` as FP16 [count, 16, 4, 64] each."""
    index = cache.storage.get_device()
    count = blocks.numel()
    blocks_ptr = _int_list(index, "blocks", blocks, count)
    flag = _int_list(index, "error_flag", error_flag, 1)
    key = torch.empty(count, _BLOCK_TOKENS, _KV_HEADS, _HEAD_DIM, dtype=_HALF, device=blocks.device)
    value = torch.empty_like(key)
    if count:
        _call(index, lib.pkv_int4_read_blocks, *cache._args(), layer, blocks_ptr, count, key.data_ptr(),
              value.data_ptr(), flag)
    return key, value


@functools.lru_cache(maxsize=4096)
def decode_plan(device_index: int, batch: int, total_blocks: int) -> tuple[int, int]:
    """Grid and workspace bytes of the decode attention (``pkv_int4_decode_plan``)."""
    grid, workspace = ctypes.c_int32(), ctypes.c_int64()
    check(lib.pkv_int4_decode_plan(device_index, batch, total_blocks, ctypes.byref(grid), ctypes.byref(workspace)))
    return grid.value, workspace.value


def decode_workspace_bytes(batch: int, grid: int) -> int:
    """Workspace of a decode launch with ``grid`` pieces (split partials; none for one piece)."""
    return (batch + grid) * _QUERY_HEADS * (_HEAD_DIM + 2) * 4 if grid > 1 else 0


def _within(rows: Tensor, out: Tensor) -> bool:
    """Whether FP16 ``rows`` [rows, heads, 64] lie where ``out`` [rows, 32, 64] is written, other than as the same rows."""
    first, begin = rows.data_ptr(), out.data_ptr()
    if first == begin and rows.shape == out.shape and rows.stride() == out.stride():
        return False
    last = first + 2 * ((rows.shape[0] - 1) * rows.stride(0) + rows.shape[1] * _HEAD_DIM)
    end = begin + 2 * ((out.shape[0] - 1) * out.stride(0) + _QUERY_HEADS * _HEAD_DIM)
    return begin < last and first < end


def _plan(index: int, query: Tensor, total_blocks: int) -> tuple[int, int, int, int]:
    """Batch, grid and the workspace of a decode launch (kept alive by the allocator until the stream passes it)."""
    batch = query.shape[0]
    _fits("batch", batch)
    _fits("total_blocks", total_blocks)
    grid, nbytes = decode_plan(index, batch, total_blocks)
    return batch, grid, nbytes, torch.empty(nbytes, dtype=_BYTE, device=query.device) if nbytes else None


def decode_attention(
    cache: Int4Cache,
    layer: int,
    query: Tensor,
    lengths: Tensor,
    prefix: Tensor,
    flat: Tensor,
    total_blocks: int,
    error_flag: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """``kernels.decode_attention`` over the 4-bit cache: rotated FP16 query [B, 32, 64].

    lengths int32 [B], prefix int32 [B + 1] (cumulative block counts) and flat
    int32 [total_blocks] (the concatenated block tables) on the device.  A row
    may have any number of tokens; one without gives zeros.
    """
    index = cache.storage.get_device()
    given = out
    query, query_stride, out, out_stride = _query_and_out(query, out, index, "batch")
    if given is not None and _within(query, out):
        query, query_stride = _dense(query), _ROW
    batch, grid, nbytes, workspace = _plan(index, query, total_blocks)
    _call(
        index, lib.pkv_int4_decode_attention, *cache._args(), layer, query.data_ptr(), query_stride,
        _int_list(index, "lengths", lengths, batch), _int_list(index, "prefix", prefix, batch + 1),
        _int_list(index, "flat", flat, total_blocks), batch, total_blocks, grid, out.data_ptr(), out_stride,
        None if workspace is None else workspace.data_ptr(), nbytes, _int_list(index, "error_flag", error_flag, 1),
    )
    return out


def decode_layer(
    cache: Int4Cache,
    layer: int,
    query: Tensor,
    key: Tensor,
    value: Tensor,
    rope_table: Tensor,
    lengths: Tensor,
    prefix: Tensor,
    flat: Tensor,
    total_blocks: int,
    error_flag: Tensor,
    out: Tensor | None = None,
    norms: HeadNorms | None = None,
) -> Tensor:
    """``kernels.decode_layer`` over the 4-bit cache, with ``norms`` after a norm of each query and key head.

    The new token of each row sits at position lengths - 1 in the row's last
    block: its K (normed, rotated) and V [B, 4, 64] are written, query [B, 32, 64]
    is normed and rotated, and attends to all of the row's tokens.  No two rows
    may share a last block.  A row without blocks gives zeros.
    """
    index = cache.storage.get_device()
    given = out
    query, query_stride, out, out_stride = _query_and_out(query, out, index, "batch")
    batch, grid, nbytes, workspace = _plan(index, query, total_blocks)
    shape = (batch, _KV_HEADS, _HEAD_DIM)
    _attention_rows("key", key, shape, index)
    _attention_rows("value", value, shape, index)
    rope = _check_rope(index, rope_table)
    key, value, strides = _aligned_pair(key, value)
    if given is not None:  # an output that lies over the inputs: rows are written while others are still read
        if _within(query, out):
            query, query_stride = _dense(query), _ROW
        if _within(key, out) or _within(value, out):
            key, value = _dense(key), _dense(value)
            strides = key.stride()
    _call(
        index, lib.pkv_int4_decode_layer, *cache._args(), layer, query.data_ptr(), query_stride, key.data_ptr(),
        value.data_ptr(), strides[0], rope, *(_NO_NORMS if norms is None else norms._args(cache)),
        _int_list(index, "lengths", lengths, batch), _int_list(index, "prefix", prefix, batch + 1),
        _int_list(index, "flat", flat, total_blocks), batch, total_blocks, grid, 1, out.data_ptr(), out_stride,
        None if workspace is None else workspace.data_ptr(), nbytes, _int_list(index, "error_flag", error_flag, 1),
    )
    return out


_PREFILL_BLOCK_BYTES = 2 * _BLOCK_TOKENS * _KV_HEADS * _HEAD_DIM * 2 + 4  # an FP16 block and its table entry


def prefill_attention(
    cache: Int4Cache,
    layer: int,
    query: Tensor,
    blocks: Tensor,
    start: int,
    error_flag: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """``kernels.prefill_attention`` over the 4-bit cache: rotated query [T, 32, 64], FP16 or FP32.

    Token t attends to positions 0 .. start + t through ``blocks`` (int32, the
    request's physical block per 16 positions).  A V group that is NaN may also
    reach tokens up to 63 positions before it (their weight for it is 0).
    """
    index = cache.storage.get_device()
    query, query_stride, out, out_stride = _query_and_out(query, out, index, "tokens", fp32=True)
    tokens = query.shape[0]
    if type(start) is not int or start < 0 or start + tokens > 2048:
        raise ValueError("the chunk must hold 1 or more tokens at positions below 2048")
    count = -(-(start + tokens) // _BLOCK_TOKENS)
    blocks_ptr = _int_list(index, "blocks", blocks, count)
    workspace = torch.empty(count * _PREFILL_BLOCK_BYTES, dtype=_BYTE, device=out.device)
    _call(index, lib.pkv_int4_prefill_attention, *cache._args(), layer, query.data_ptr(), query.dtype is _FLOAT,
          query_stride, blocks_ptr, start, tokens, out.data_ptr(), out_stride, workspace.data_ptr(),
          count * _PREFILL_BLOCK_BYTES, _int_list(index, "error_flag", error_flag, 1))
    return out
