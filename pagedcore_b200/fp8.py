"""8-bit decode path: E4M3 rows, weights and KV cache, and the operators over them.

The 8-bit forms of the FP16 operators in :mod:`pagedcore_b200.kernels`, in the
same manner (tensor checks here, work in the sm_100a kernels, the current CUDA
stream of the tensors' device):

- ``add_rms_norm``, ``silu_mul`` and ``quantize_rows`` make :class:`Fp8Rows`,
  codes with one scale per row and 128 values;
- ``linear`` multiplies them by an :class:`Fp8Weight` (a scale per 128 x 128
  block, from ``quantize_weight`` or a checkpoint);
- ``append_kv``, ``decode_layer``, ``decode_attention``, ``prefill_attention``
  and ``read_blocks`` work on an :class:`Fp8Cache`, a scale per block of 16
  tokens and head.

Scales made here are powers of two, so every stored value is an FP16 number.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
from dataclasses import dataclass

import torch
from torch import Tensor

from pagedcore_b200._lib import check, lib
from pagedcore_b200.kernels import linear_error_flag

GROUP = 128  # values per scale of rows; both sides of a weight's blocks
_KV_HEADS = 4
_QUERY_HEADS = 32
_HEAD_DIM = 64
_BLOCK_TOKENS = 16
_CODES = torch.float8_e4m3fn


def _groups(width: int) -> int:
    return -(-width // GROUP)


def _device(*tensors: Tensor) -> torch.device:
    """The CUDA device that every tensor is on."""
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError("8-bit operators need CUDA tensors")
    for tensor in tensors:
        if tensor.device != device:
            raise ValueError(f"every tensor must be on {device}")
    return device


@contextlib.contextmanager
def _switched(device: torch.device):
    with torch.cuda.device(device):
        yield


_SAME = contextlib.nullcontext()


def _on(device: torch.device):
    """Launch on ``device`` whatever the current device is."""
    return _SAME if torch.cuda.current_device() == device.index else _switched(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


@dataclass(frozen=True, slots=True)
class Fp8Rows:
    """E4M3 codes [rows, width] and FP32 scales [rows, ceil(width / 128)]."""

    codes: Tensor
    scales: Tensor

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)

    def to_half(self, out: Tensor | None = None) -> Tensor:
        """The values as FP16 [rows, width] (exact for scales made by this module)."""
        _check_rows(self)
        rows, width = self.codes.shape
        device = _device(self.codes, self.scales)
        if not self.codes.is_contiguous():
            raise ValueError("to_half needs contiguous codes")
        if out is None:
            out = torch.empty((rows, width), dtype=torch.float16, device=device)
        elif out.shape != (rows, width) or out.dtype != torch.float16 or out.stride(1) != 1 or out.device != device:
            raise ValueError(f"out must be FP16 [{rows}, {width}] with contiguous rows")
        if rows == 0:
            return out
        with _on(device):
            check(lib.pkv_fp8_to_half(self.codes.data_ptr(), self.scales.data_ptr(), rows, width, out.data_ptr(),
                                      out.stride(0), _stream(device)))
        return out


@dataclass(frozen=True, slots=True)
class Fp8Weight:
    """E4M3 codes [n, k] and FP32 scales [ceil(n / 128), ceil(k / 128)]."""

    codes: Tensor
    scales: Tensor

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)


def _check_rows(x: Fp8Rows) -> None:
    codes, scales = x.codes, x.scales
    if codes.ndim != 2 or codes.dtype != _CODES or (codes.numel() and codes.stride(1) != 1):
        raise ValueError("8-bit rows must be E4M3 [rows, width] with contiguous rows")
    if (
        scales.shape != (codes.shape[0], _groups(codes.shape[1]))
        or scales.dtype != torch.float32
        or not scales.is_contiguous()
    ):
        raise ValueError("8-bit rows need contiguous FP32 scales [rows, ceil(width / 128)]")


def _empty_rows(rows: int, width: int, device: torch.device) -> Fp8Rows:
    return Fp8Rows(
        torch.empty((rows, width), dtype=_CODES, device=device),
        torch.empty((rows, _groups(width)), dtype=torch.float32, device=device),
    )


def _half_matrix(name: str, tensor: Tensor, shape: tuple[int, ...]) -> None:
    if tensor.shape != shape or tensor.dtype != torch.float16 or not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous FP16 {list(shape)}")


def add_rms_norm(
    hidden: Tensor,
    delta: Tensor | None,
    weight: Tensor,
    *,
    residual: Tensor | None = None,
    eps: float = 1e-5,
) -> Fp8Rows:
    """``kernels.add_rms_norm`` with an 8-bit output.

    hidden, delta FP16 [rows, dim], weight FP16 [dim].  With ``delta`` the sum
    is written as FP16 to ``residual`` (``hidden`` itself by default); the
    norm is taken of the unrounded sum, in FP32, and rounded once, to E4M3.
    """
    if hidden.ndim != 2:
        raise ValueError("hidden must be contiguous FP16 [rows, dim]")
    rows, dim = hidden.shape
    _half_matrix("hidden", hidden, (rows, dim))
    _half_matrix("weight", weight, (dim,))
    if delta is None:
        device = _device(hidden, weight)
        delta_ptr = residual_ptr = None
    else:
        if residual is None:
            residual = hidden
        _half_matrix("delta", delta, (rows, dim))
        _half_matrix("residual", residual, (rows, dim))
        device = _device(hidden, weight, delta, residual)
        delta_ptr, residual_ptr = delta.data_ptr(), residual.data_ptr()
    out = _empty_rows(rows, dim, device)
    if rows == 0:
        return out
    with _on(device):
        check(lib.pkv_fp8_add_rms_norm(hidden.data_ptr(), delta_ptr, weight.data_ptr(), residual_ptr,
                                       out.codes.data_ptr(), out.scales.data_ptr(), rows, dim, eps, _stream(device)))
    return out


def _quantize(x: Tensor, width: int, silu_pairs: bool) -> Fp8Rows:
    device = _device(x)
    out = _empty_rows(x.shape[0], width, device)
    if x.shape[0] == 0:
        return out
    with _on(device):
        check(lib.pkv_fp8_quantize(x.data_ptr(), max(x.stride(0), x.shape[1]), silu_pairs, x.shape[0], width,
                                   out.codes.data_ptr(), out.scales.data_ptr(), _stream(device)))
    return out


def quantize_rows(x: Tensor) -> Fp8Rows:
    """FP16 [rows, width] (rows contiguous, any row stride that is a multiple of 8) as 8-bit rows."""
    if x.ndim != 2 or x.dtype != torch.float16 or (x.numel() and x.stride(1) != 1):
        raise ValueError("x must be FP16 [rows, width] with contiguous rows")
    return _quantize(x, x.shape[1], False)


def silu_mul(gate_up: Tensor) -> Fp8Rows:
    """``silu(gate) * up`` of FP16 [rows, 2 * inter] (gate first) as 8-bit rows, rounded once."""
    if gate_up.ndim != 2 or gate_up.dtype != torch.float16 or gate_up.shape[1] % 2 or not gate_up.is_contiguous():
        raise ValueError("gate_up must be contiguous FP16 [rows, 2 * inter]")
    return _quantize(gate_up, gate_up.shape[1] // 2, True)


def quantize_weight(weight: Tensor) -> Fp8Weight:
    """A floating [n, k] weight as codes and a scale per 128 x 128 block (once, at load time)."""
    if weight.ndim != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a floating [n, k] matrix")
    n, k = weight.shape
    tall, wide = _groups(n), _groups(k)
    padded = torch.zeros((tall * GROUP, wide * GROUP), dtype=torch.float32, device=weight.device)
    padded[:n, :k] = weight.detach().float()
    blocks = padded.view(tall, GROUP, wide, GROUP)
    mantissa, exponent = torch.frexp(blocks.abs().amax((1, 3)))
    exponent = (exponent - 9 + (mantissa > 0.875).int()).clamp(-15, 8)  # 448 = 0.875 * 2^9
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    scaled = (blocks / scales[:, None, :, None]).clamp(-448.0, 448.0).to(_CODES)
    codes = scaled.view(torch.uint8).reshape(tall * GROUP, wide * GROUP)[:n, :k].contiguous().view(_CODES)
    return Fp8Weight(codes, scales.contiguous())


def linear(x: Fp8Rows, weight: Fp8Weight, out: Tensor | None = None) -> Tensor:
    """``kernels.linear`` for 8-bit rows [rows, k] and weight [n, k]: FP16 [rows, n].

    Any number of rows and any n; k a multiple of 16.  FP32 sums on the
    tensor cores, scaled block by block, rounded once.
    """
    _check_rows(x)
    (rows, k), (n, wk) = x.codes.shape, weight.codes.shape
    if wk != k or weight.codes.dtype != _CODES or not weight.codes.is_contiguous():
        raise ValueError(f"weight must be contiguous E4M3 [n, {k}]")
    if (
        weight.scales.shape != (_groups(n), _groups(k))
        or weight.scales.dtype != torch.float32
        or not weight.scales.is_contiguous()
    ):
        raise ValueError("weight needs contiguous FP32 scales [ceil(n / 128), ceil(k / 128)]")
    device = _device(x.codes, x.scales, weight.codes, weight.scales)
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float16, device=device)
    elif out.shape != (rows, n) or out.dtype != torch.float16 or out.stride(1) != 1 or out.device != device:
        raise ValueError(f"out must be FP16 [{rows}, {n}] with contiguous rows")
    if rows == 0:
        return out
    with _on(device):
        check(lib.pkv_fp8_linear(x.codes.data_ptr(), max(x.codes.stride(0), k), x.scales.data_ptr(),
                                 weight.codes.data_ptr(), weight.scales.data_ptr(), rows, n, k, out.data_ptr(),
                                 max(out.stride(0), n), linear_error_flag(device).data_ptr(), _stream(device)))
    return out


# -- the KV cache ------------------------------------------------------------------


@dataclass(frozen=True, slots=True)
class Fp8Cache:
    """An 8-bit KV cache: E4M3 codes and FP32 scales.

    key_codes [layers, blocks, 4, 16, 64], value_codes [layers, blocks, 4, 64, 16]
    (V is held transposed), key_scales and value_scales [layers, blocks, 4].
    A slot id is physical_block * 16 + slot_in_block, as in the FP16 pool.
    """

    key_codes: Tensor
    value_codes: Tensor
    key_scales: Tensor
    value_scales: Tensor

    def __post_init__(self) -> None:
        codes = self.key_codes
        if codes.ndim != 5 or codes.shape[2:] != (_KV_HEADS, _BLOCK_TOKENS, _HEAD_DIM):
            raise ValueError("key_codes must be E4M3 [layers, blocks, 4, 16, 64]")
        layers, blocks = codes.shape[:2]
        if layers < 1 or blocks < 1:
            raise ValueError("an 8-bit cache needs at least one layer and one block")
        if self.value_codes.shape != (layers, blocks, _KV_HEADS, _HEAD_DIM, _BLOCK_TOKENS):
            raise ValueError("value_codes must be E4M3 [layers, blocks, 4, 64, 16]")
        for tensor in (codes, self.value_codes):
            if tensor.dtype != _CODES or not tensor.is_contiguous():
                raise ValueError("cache codes must be contiguous E4M3 storage")
        for tensor in (self.key_scales, self.value_scales):
            if tensor.shape != (layers, blocks, _KV_HEADS) or tensor.dtype != torch.float32 or not tensor.is_contiguous():
                raise ValueError("cache scales must be contiguous FP32 [layers, blocks, 4]")
        _device(codes, self.value_codes, self.key_scales, self.value_scales)

    @classmethod
    def empty(cls, layers: int, blocks: int, device: str | torch.device = "cuda") -> Fp8Cache:
        """Uninitialised storage: only written, valid slots may be read."""
        return cls(
            torch.empty((layers, blocks, _KV_HEADS, _BLOCK_TOKENS, _HEAD_DIM), dtype=_CODES, device=device),
            torch.empty((layers, blocks, _KV_HEADS, _HEAD_DIM, _BLOCK_TOKENS), dtype=_CODES, device=device),
            torch.empty((layers, blocks, _KV_HEADS), dtype=torch.float32, device=device),
            torch.empty((layers, blocks, _KV_HEADS), dtype=torch.float32, device=device),
        )

    @property
    def device(self) -> torch.device:
        return self.key_codes.device

    @property
    def layers(self) -> int:
        return self.key_codes.shape[0]

    @property
    def num_blocks(self) -> int:
        return self.key_codes.shape[1]

    def _args(self) -> tuple[int, int, int, int, int, int]:
        shape = self.key_codes.shape
        return (self.key_codes.data_ptr(), self.value_codes.data_ptr(), self.key_scales.data_ptr(),
                self.value_scales.data_ptr(), shape[0], shape[1])


def _require(device: torch.device, dtype: torch.dtype, **tensors: Tensor) -> None:
    for name, tensor in tensors.items():
        if tensor.device != device or tensor.dtype != dtype:
            raise ValueError(f"{name} must be {dtype} on {device}")


def _int_list(device: torch.device, name: str, tensor: Tensor, count: int) -> None:
    if tensor.device != device or tensor.dtype != torch.int32 or not tensor.is_contiguous() or tensor.numel() < count:
        raise ValueError(f"{name} must hold {count} contiguous int32 values on {device}")


def _check_flag(device: torch.device, error_flag: Tensor) -> None:
    _int_list(device, "error_flag", error_flag, 1)


def _check_rope(device: torch.device, table: Tensor) -> None:
    _require(device, torch.float16, rope_table=table)
    if table.shape != (2, 2048, 32) or not table.is_contiguous():
        raise ValueError("rope_table must be contiguous FP16 [2, 2048, 32]")


def _rows_ok(tensor: Tensor) -> bool:
    """Inner [heads, 64] contiguous and rows 16-byte aligned."""
    return (
        tensor.stride()[-2:] == (_HEAD_DIM, 1)
        and all(stride % 8 == 0 for stride in tensor.stride()[:-2])
        and tensor.data_ptr() % 16 == 0
    )


def append_kv(
    cache: Fp8Cache,
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
) -> Tensor | None:
    """Write FP16 K/V [layers, tokens, 4, 64] into the cache at ``slots`` (int32 [tokens]).

    With ``rope_table`` K is rotated at ``positions`` first, and ``query``
    [layers, tokens, 32, 64] is returned rotated (in ``query_out`` when given,
    which may be ``query`` itself).  The tokens of one block must be
    consecutive, in the list and in the block, as a request's positions are.
    """
    device = cache.device
    if key.ndim != 4 or key.shape[2:] != (_KV_HEADS, _HEAD_DIM) or value.shape != key.shape:
        raise ValueError("K and V must share FP16 [layers, tokens, 4, 64]")
    _require(device, torch.float16, key=key, value=value)
    layers, tokens = key.shape[:2]
    _int_list(device, "slots", slots, tokens)
    _check_flag(device, error_flag)
    if (rope_table is None) != (positions is None) or (query is not None and rope_table is None):
        raise ValueError("rope_table goes with positions, query with both")
    if rope_table is not None:
        _check_rope(device, rope_table)
        _int_list(device, "positions", positions, tokens)
    if layers == 0 or tokens == 0:
        return query
    if not (_rows_ok(key) and value.stride() == key.stride() and _rows_ok(value)):
        key, value = key.contiguous(), value.contiguous()
    q_ptr = out_ptr = None
    q_strides = out_strides = (0, 0)
    if query is not None:
        if query.shape != (layers, tokens, _QUERY_HEADS, _HEAD_DIM):
            raise ValueError("query must be FP16 [layers, tokens, 32, 64]")
        _require(device, torch.float16, query=query)
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=torch.float16, device=device)
        elif query_out.shape != query.shape or not _rows_ok(query_out):
            raise ValueError("query_out must be FP16 [layers, tokens, 32, 64] with contiguous, 16-byte aligned rows")
        _require(device, torch.float16, query_out=query_out)
        if not _rows_ok(query):
            query = query.contiguous()
        q_ptr, out_ptr = query.data_ptr(), query_out.data_ptr()
        q_strides, out_strides = query.stride()[:2], query_out.stride()[:2]
    with _on(device):
        check(
            lib.pkv_fp8_append_kv(
                *cache._args(), layer_begin, layers, key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1),
                slots.data_ptr(), None if positions is None else positions.data_ptr(), tokens,
                None if rope_table is None else rope_table.data_ptr(), q_ptr, *q_strides, out_ptr, *out_strides,
                error_flag.data_ptr(), _stream(device),
            )
        )
    return query_out


def read_blocks(cache: Fp8Cache, layer: int, blocks: Tensor, error_flag: Tensor) -> tuple[Tensor, Tensor]:
    """K and V of ``blocks`` (int32 [count]) at ``layer`` as FP16 [count, 16, 4, 64] each."""
    device = cache.device
    count = blocks.numel()
    _int_list(device, "blocks", blocks, count)
    _check_flag(device, error_flag)
    out = torch.empty((2, count, _BLOCK_TOKENS, _KV_HEADS, _HEAD_DIM), dtype=torch.float16, device=device)
    if count == 0:
        return out[0], out[1]
    with _on(device):
        check(lib.pkv_fp8_read_blocks(*cache._args(), layer, blocks.data_ptr(), count, out.data_ptr(), out.stride(0),
                                      error_flag.data_ptr(), _stream(device)))
    return out[0], out[1]


@functools.lru_cache(maxsize=4096)
def decode_plan(device_index: int, batch: int, total_blocks: int) -> tuple[int, int]:
    """Grid and workspace bytes of the decode attention (``pkv_fp8_decode_plan``)."""
    grid, workspace = ctypes.c_int32(), ctypes.c_int64()
    check(lib.pkv_fp8_decode_plan(device_index, batch, total_blocks, ctypes.byref(grid), ctypes.byref(workspace)))
    return grid.value, workspace.value


def decode_workspace_bytes(batch: int, grid: int) -> int:
    """Workspace of a decode launch with ``grid`` pieces (rotated queries, then split partials)."""
    return batch * _QUERY_HEADS * _HEAD_DIM * 2 + (batch + grid) * _QUERY_HEADS * (_HEAD_DIM + 2) * 4


def _attention_rows(name: str, tensor: Tensor, shape: tuple[int, ...], device: torch.device) -> None:
    if tensor.shape != shape or tensor.dtype != torch.float16 or tensor.device != device:
        raise ValueError(f"{name} must be FP16 {list(shape)} on {device}")


def _decode(cache, layer, query, new, rope_table, lengths, prefix, flat, total_blocks, error_flag, out) -> Tensor:
    device = cache.device
    if query.ndim != 3 or query.shape[0] < 1:
        raise ValueError("query must be FP16 [batch, 32, 64] of a nonempty batch")
    batch = query.shape[0]
    _attention_rows("query", query, (batch, _QUERY_HEADS, _HEAD_DIM), device)
    if not _rows_ok(query) or query.stride(0) < _QUERY_HEADS * _HEAD_DIM:
        query = query.contiguous()
    if out is None:
        out = torch.empty((batch, _QUERY_HEADS, _HEAD_DIM), dtype=torch.float16, device=device)
    else:
        _attention_rows("out", out, (batch, _QUERY_HEADS, _HEAD_DIM), device)
        if not _rows_ok(out):
            raise ValueError("out must be FP16 [batch, 32, 64] with contiguous, 16-byte aligned rows")
    _int_list(device, "lengths", lengths, batch)
    _int_list(device, "prefix", prefix, batch + 1)
    _int_list(device, "flat", flat, total_blocks)
    _check_flag(device, error_flag)
    grid, workspace_bytes = decode_plan(device.index, batch, total_blocks)
    workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=device)
    tables = (lengths.data_ptr(), prefix.data_ptr(), flat.data_ptr(), batch, total_blocks, grid, out.data_ptr(),
              max(out.stride(0), _QUERY_HEADS * _HEAD_DIM), workspace.data_ptr(), workspace_bytes,
              error_flag.data_ptr())
    query_stride = max(query.stride(0), _QUERY_HEADS * _HEAD_DIM)
    with _on(device):
        if new is None:
            check(lib.pkv_fp8_decode_attention(*cache._args(), layer, query.data_ptr(), query_stride, *tables,
                                               _stream(device)))
        else:
            key, value = new
            check(lib.pkv_fp8_decode_layer(*cache._args(), layer, query.data_ptr(), query_stride, key.data_ptr(),
                                           value.data_ptr(), key.stride(0), rope_table.data_ptr(), *tables,
                                           _stream(device)))
    return out


def decode_attention(
    cache: Fp8Cache,
    layer: int,
    query: Tensor,
    lengths: Tensor,
    prefix: Tensor,
    flat: Tensor,
    total_blocks: int,
    error_flag: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """``kernels.decode_attention`` over the 8-bit cache: rotated FP16 query [B, 32, 64].

    lengths int32 [B], prefix int32 [B + 1] (cumulative block counts) and flat
    int32 [total_blocks] (the concatenated block tables) on the device.  A row
    without tokens gives zeros.
    """
    return _decode(cache, layer, query, None, None, lengths, prefix, flat, total_blocks, error_flag, out)


def decode_layer(
    cache: Fp8Cache,
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
) -> Tensor:
    """``kernels.decode_layer`` over the 8-bit cache.

    The new token of each row sits at position lengths - 1 in the row's last
    block: its K (rotated) and V [B, 4, 64] are written, query [B, 32, 64] is
    rotated, and attends to all of the row's tokens.  No two rows may share
    a last block.
    """
    device = cache.device
    batch = query.shape[0]
    _attention_rows("key", key, (batch, _KV_HEADS, _HEAD_DIM), device)
    _attention_rows("value", value, (batch, _KV_HEADS, _HEAD_DIM), device)
    _check_rope(device, rope_table)
    if not (_rows_ok(key) and value.stride() == key.stride() and _rows_ok(value)):
        key, value = key.contiguous(), value.contiguous()
    return _decode(cache, layer, query, (key, value), rope_table, lengths, prefix, flat, total_blocks, error_flag, out)


_PREFILL_BLOCK_BYTES = 2 * _BLOCK_TOKENS * _KV_HEADS * _HEAD_DIM * 2 + 4  # an FP16 block and its table entry


def prefill_attention(
    cache: Fp8Cache,
    layer: int,
    query: Tensor,
    blocks: Tensor,
    start: int,
    error_flag: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """``kernels.prefill_attention`` over the 8-bit cache: rotated FP16 query [T, 32, 64].

    Token t attends to positions 0 .. start + t through ``blocks`` (int32, the
    request's physical block per 16 positions).
    """
    device = cache.device
    if query.ndim != 3 or query.shape[0] < 1:
        raise ValueError("query must be FP16 [tokens, 32, 64]")
    tokens = query.shape[0]
    _attention_rows("query", query, (tokens, _QUERY_HEADS, _HEAD_DIM), device)
    if type(start) is not int or start < 0 or start + tokens > 2048:
        raise ValueError("the chunk must hold 1 or more tokens at positions below 2048")
    count = -(-(start + tokens) // _BLOCK_TOKENS)
    _int_list(device, "blocks", blocks, count)
    _check_flag(device, error_flag)
    if not _rows_ok(query) or query.stride(0) < _QUERY_HEADS * _HEAD_DIM:
        query = query.contiguous()
    if out is None:
        out = torch.empty((tokens, _QUERY_HEADS, _HEAD_DIM), dtype=torch.float16, device=device)
    else:
        _attention_rows("out", out, (tokens, _QUERY_HEADS, _HEAD_DIM), device)
        if not _rows_ok(out):
            raise ValueError("out must be FP16 [tokens, 32, 64] with contiguous, 16-byte aligned rows")
    workspace = torch.empty(count * _PREFILL_BLOCK_BYTES, dtype=torch.uint8, device=device)
    with _on(device):
        check(lib.pkv_fp8_prefill_attention(*cache._args(), layer, query.data_ptr(),
                                            max(query.stride(0), _QUERY_HEADS * _HEAD_DIM), blocks.data_ptr(), start,
                                            tokens, out.data_ptr(), max(out.stride(0), _QUERY_HEADS * _HEAD_DIM),
                                            workspace.data_ptr(), workspace.numel(), error_flag.data_ptr(),
                                            _stream(device)))
    return out
