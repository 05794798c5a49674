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
A token takes 288 bytes a layer, FP16 1024 and E4M3 514.

With :class:`HeadNorms`, queries and keys are normed head by head before they
are rotated, in the same pass.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch
from torch import Tensor

from pagedcore_b200 import build
from pagedcore_b200._lib import check, lib

try:
    from pagedcore_b200 import _int4_ops

    _built_for = getattr(_int4_ops, "built_for", "an earlier form of this package")
    if _built_for != build.built_for():
        raise ImportError(f"it was built for {_built_for}, not for {build.built_for()}")
except ImportError as error:
    raise ImportError(
        "pagedcore_b200/_int4_ops.so is missing or was built for another torch or Python: "
        "build it with `python -m pagedcore_b200.build`"
    ) from error

BLOCK_BYTES = 4608  # of 16 tokens in one layer
_QUERY_HEADS = 32
_HEAD_DIM = 64


@dataclass(frozen=True, slots=True)
class Int4Cache:
    """A 4-bit KV cache: bytes [layers, blocks, 4608].  Its tensor is checked once and stays.

    A block holds 16 tokens: for each of the 4 heads 512 bytes of K codes [4 groups,
    16 tokens, 8], 512 of V codes [8 chunks of 8 dims, 16 tokens, 4], 64 of K scales
    [4 groups, 16 tokens] and 64 of V scales (``include/pagedkv.h`` gives the order of
    the codes).  A slot id is physical_block * 16 + slot_in_block, as in the FP16 pool.
    """

    storage: Tensor

    def __post_init__(self) -> None:
        _int4_ops.check_cache(self.storage)

    @classmethod
    def empty(cls, layers: int, blocks: int, device: str | torch.device = "cuda") -> Int4Cache:
        """Uninitialised storage: only written, valid slots may be read."""
        return cls(torch.empty((layers, blocks, BLOCK_BYTES), dtype=torch.uint8, device=device))

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


@dataclass(frozen=True, slots=True)
class HeadNorms:
    """Weights of the RMS norms of each query and key head, FP16 [layers, 64] each, for a cache's layers.

    x * rsqrt(mean(x^2) + eps) * weight over the 64 dims of a head, before the rotation.  An allocator
    and its step graphs keep the weights' addresses: values may change in place, the tensors stay.
    """

    query: Tensor
    key: Tensor
    eps: float = 1e-5

    def check(self, cache: Int4Cache) -> None:
        """Raise ValueError unless these are norms for the layers of ``cache``."""
        _int4_ops.check_norms(cache.storage, self.query, self.key, self.eps)


def overlaps(rows: Tensor, out: Tensor) -> bool:
    """Whether ``rows`` [rows, heads, 64] lie where ``out`` [rows, 32, 64] is written, other than as the same rows."""
    return _int4_ops.overlaps(rows, out)


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
    if norms is None:
        return _int4_ops.append_kv(
            cache.storage, key, value, slots, layer_begin, error_flag, positions, rope_table, query, query_out, None, None,
            0.0,
        )
    return _int4_ops.append_kv(
        cache.storage, key, value, slots, layer_begin, error_flag, positions, rope_table, query, query_out, norms.query,
        norms.key, norms.eps,
    )


def read_blocks(cache: Int4Cache, layer: int, blocks: Tensor, error_flag: Tensor) -> tuple[Tensor, Tensor]:
    """K and V of ``blocks`` (int32 [count]) at ``layer`` as FP16 [count, 16, 4, 64] each."""
    return _int4_ops.read_blocks(cache.storage, layer, blocks, error_flag)


@functools.lru_cache(maxsize=4096)
def decode_plan(device_index: int, batch: int, total_blocks: int) -> tuple[int, int]:
    """Grid and workspace bytes of the decode attention (``pkv_int4_decode_plan``)."""
    grid, workspace = ctypes.c_int32(), ctypes.c_int64()
    check(lib.pkv_int4_decode_plan(device_index, batch, total_blocks, ctypes.byref(grid), ctypes.byref(workspace)))
    return grid.value, workspace.value


def decode_workspace_bytes(batch: int, grid: int) -> int:
    """Workspace of a decode launch with ``grid`` pieces (split partials; none for one piece)."""
    return (batch + grid) * _QUERY_HEADS * (_HEAD_DIM + 2) * 4 if grid > 1 else 0


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
    return _int4_ops.decode_attention(
        cache.storage, layer, query, lengths, prefix, flat, total_blocks, error_flag, out
    )


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
    if norms is None:
        return _int4_ops.decode_layer(
            cache.storage, layer, query, key, value, rope_table, lengths, prefix, flat, total_blocks, error_flag, out,
            None, None, 0.0,
        )
    return _int4_ops.decode_layer(
        cache.storage, layer, query, key, value, rope_table, lengths, prefix, flat, total_blocks, error_flag, out,
        norms.query, norms.key, norms.eps,
    )


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
    return _int4_ops.prefill_attention(cache.storage, layer, query, blocks, start, error_flag, out)
