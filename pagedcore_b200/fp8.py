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
_HALF = torch.float16
_FLOAT = torch.float32
_INT = torch.int32
_ROW = _QUERY_HEADS * _HEAD_DIM  # values of a query row
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


_MOST = 2**31 - 2**16  # rows, columns and list entries: the C ABI's int32, and a step of a row loop


def _fits(name: str, count: int) -> None:
    """``count`` as the kernels take it (ctypes would cut it to 32 bits without a word)."""
    if count > _MOST:
        raise ValueError(f"{name} must be at most {_MOST}, not {count}")


def _groups(width: int) -> int:
    return -(-width // GROUP)


def _device(first: Tensor, *others: Tensor) -> int:
    """Index of the CUDA device that every tensor is on."""
    index = first.get_device()
    if index < 0:
        raise ValueError("8-bit operators need CUDA tensors")
    for tensor in others:
        if tensor.get_device() != index:
            raise ValueError(f"every tensor must be on cuda:{index}")
    return index


def _call(index: int, function, *args) -> None:
    """Launch on device ``index`` and its current stream, whatever the current device is.

    The raw stream handle spares the Stream object that
    ``torch.cuda.current_stream`` builds (2 us of a 5 us call).
    """
    if _current_device() == index:
        status = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, _raw_stream(index))
    if status:
        check(status)


def _row_stride(name: str, tensor: Tensor, width: int) -> int:
    """Row stride of a matrix whose rows must not overlap (one row's may be anything)."""
    stride = tensor.stride(0)
    if stride >= width:
        return stride
    if tensor.shape[0] > 1:
        raise ValueError(f"the rows of {name} overlap")
    return width


@dataclass(slots=True)
class Fp8Rows:
    """E4M3 codes [rows, width] and FP32 scales [rows, ceil(width / 128)]."""

    codes: Tensor
    scales: Tensor

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)

    def to_half(self, out: Tensor | None = None) -> Tensor:
        """The values as FP16 [rows, width] (exact for scales made by this module)."""
        rows, width = _check_rows(self)
        codes, scales = self.codes, self.scales
        index = _device(codes, scales)
        if not codes.is_contiguous():
            raise ValueError("to_half needs contiguous codes")
        if out is None:
            out = torch.empty_like(codes, dtype=_HALF)
            stride = width
        else:
            if out.shape != (rows, width) or out.dtype is not _HALF or out.stride(1) != 1 or out.get_device() != index:
                raise ValueError(f"out must be FP16 [{rows}, {width}] with contiguous rows")
            stride = _row_stride("out", out, width)
        if rows:
            _call(index, lib.pkv_fp8_to_half, codes.data_ptr(), scales.data_ptr(), rows, width,
                  out.data_ptr(), stride)
        return out


@dataclass(slots=True)
class Fp8Weight:
    """E4M3 codes [n, k] and FP32 scales [ceil(n / 128), ceil(k / 128)]."""

    codes: Tensor
    scales: Tensor

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)


def _check_rows(x: Fp8Rows) -> tuple[int, int]:
    codes, scales = x.codes, x.scales
    shape = codes.shape
    if len(shape) != 2 or codes.dtype is not _CODES or codes.stride(1) != 1:
        raise ValueError("8-bit rows must be E4M3 [rows, width] with contiguous rows")
    rows, width = shape
    _fits("rows", rows)
    _fits("width", width)
    if scales.shape != (rows, -(-width // GROUP)) or scales.dtype is not _FLOAT or not scales.is_contiguous():
        raise ValueError("8-bit rows need contiguous FP32 scales [rows, ceil(width / 128)]")
    return rows, width


def _empty_rows(x: Tensor, rows: int, width: int) -> Fp8Rows:
    """Uninitialised 8-bit rows on the device of ``x``."""
    device = x.device  # sizes one by one: torch.empty takes a tuple 0.7 us slower
    return Fp8Rows(
        torch.empty(rows, width, dtype=_CODES, device=device),
        torch.empty(rows, -(-width // GROUP), dtype=_FLOAT, device=device),
    )


def _half_matrix(name: str, tensor: Tensor, shape: tuple[int, ...]) -> None:
    if tensor.shape != shape or tensor.dtype is not _HALF or not tensor.is_contiguous():
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
    shape = hidden.shape
    if len(shape) != 2:
        raise ValueError("hidden must be contiguous FP16 [rows, dim]")
    rows, dim = shape
    _fits("rows", rows)
    _fits("dim", dim)
    _half_matrix("hidden", hidden, shape)
    _half_matrix("weight", weight, (dim,))
    delta_ptr = residual_ptr = None
    if delta is None:
        index = _device(hidden, weight)
    else:
        if residual is None:
            residual = hidden
        else:
            _half_matrix("residual", residual, shape)
        _half_matrix("delta", delta, shape)
        index = _device(hidden, weight, delta, residual)
        delta_ptr, residual_ptr = delta.data_ptr(), residual.data_ptr()
    out = _empty_rows(hidden, rows, dim)
    if rows:
        _call(index, lib.pkv_fp8_add_rms_norm, hidden.data_ptr(), delta_ptr, weight.data_ptr(), residual_ptr,
              out.codes.data_ptr(), out.scales.data_ptr(), rows, dim, eps)
    return out


def _quantize(x: Tensor, width: int, silu_pairs: bool) -> Fp8Rows:
    rows, columns = x.shape
    _fits("rows", rows)
    _fits("width", columns)
    index = _device(x)
    out = _empty_rows(x, rows, width)
    if rows:
        _call(index, lib.pkv_fp8_quantize, x.data_ptr(), _row_stride("x", x, columns), silu_pairs, rows, width,
              out.codes.data_ptr(), out.scales.data_ptr())
    return out


def quantize_rows(x: Tensor) -> Fp8Rows:
    """FP16 [rows, width] (rows contiguous, any row stride that is a multiple of 8) as 8-bit rows.

    Any width that is a multiple of 8; ``linear`` takes those of 16.
    """
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
    finite = blocks.isfinite()
    mantissa, exponent = torch.frexp(torch.where(finite, blocks.abs(), 0.0).amax((1, 3)))
    exponent = (exponent - 9 + (mantissa > 0.875).int()).clamp(-15, 8)  # 448 = 0.875 * 2^9
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    largest = torch.where(exponent == 8, 240.0, 448.0)[:, None, :, None]  # at 2^8 the values end inside FP16
    scaled = torch.minimum(torch.maximum(blocks / scales[:, None, :, None], -largest), largest)
    scaled = torch.where(finite, scaled, torch.nan).to(_CODES)
    codes = scaled.view(torch.uint8).reshape(tall * GROUP, wide * GROUP)[:n, :k].contiguous().view(_CODES)
    return Fp8Weight(codes, scales.contiguous())


def linear(x: Fp8Rows, weight: Fp8Weight, out: Tensor | None = None) -> Tensor:
    """``kernels.linear`` for 8-bit rows [rows, k] and weight [n, k]: FP16 [rows, n].

    Any number of rows and any n; k a multiple of 16.  FP32 sums on the
    tensor cores, scaled block by block, rounded once.
    """
    rows, k = _check_rows(x)
    codes, scales = weight.codes, weight.scales
    shape = codes.shape
    if len(shape) != 2 or shape[1] != k or codes.dtype is not _CODES or not codes.is_contiguous():
        raise ValueError(f"weight must be contiguous E4M3 [n, {k}]")
    n = shape[0]
    _fits("n", n)
    if scales.shape != (_groups(n), _groups(k)) or scales.dtype is not _FLOAT or not scales.is_contiguous():
        raise ValueError("weight needs contiguous FP32 scales [ceil(n / 128), ceil(k / 128)]")
    index = _device(x.codes, x.scales, codes, scales)
    x_stride = _row_stride("x", x.codes, k)
    if out is None:
        out = torch.empty(rows, n, dtype=_HALF, device=codes.device)
        stride = n
    else:
        if out.shape != (rows, n) or out.dtype is not _HALF or out.stride(1) != 1 or out.get_device() != index:
            raise ValueError(f"out must be FP16 [{rows}, {n}] with contiguous rows")
        stride = _row_stride("out", out, n)
    if rows:
        _call(index, lib.pkv_fp8_linear, x.codes.data_ptr(), x_stride, x.scales.data_ptr(),
              codes.data_ptr(), scales.data_ptr(), rows, n, k, out.data_ptr(), stride,
              linear_error_flag(codes.device).data_ptr())
    return out


# -- the KV cache ------------------------------------------------------------------


@dataclass(slots=True)
class Fp8Cache:
    """An 8-bit KV cache: E4M3 codes and FP32 scales.

    key_codes [layers, blocks, 4, 16, 64], value_codes [layers, blocks, 4, 64, 16]
    (V is held transposed), key_scales and value_scales [layers, blocks, 4],
    powers of two from 2^-15 to 2^8 as ``append_kv`` makes them (the decode
    attention takes V's scale as an exponent).
    A slot id is physical_block * 16 + slot_in_block, as in the FP16 pool.
    """

    key_codes: Tensor
    value_codes: Tensor
    key_scales: Tensor
    value_scales: Tensor

    def __post_init__(self) -> None:
        keys, values, key_scales, value_scales = self.key_codes, self.value_codes, self.key_scales, self.value_scales
        shape = keys.shape
        if len(shape) != 5 or shape[2:] != (_KV_HEADS, _BLOCK_TOKENS, _HEAD_DIM):
            raise ValueError("key_codes must be E4M3 [layers, blocks, 4, 16, 64]")
        layers, blocks = shape[0], shape[1]
        if layers < 1 or blocks < 1:
            raise ValueError("an 8-bit cache needs at least one layer and one block")
        if values.shape != (layers, blocks, _KV_HEADS, _HEAD_DIM, _BLOCK_TOKENS):
            raise ValueError("value_codes must be E4M3 [layers, blocks, 4, 64, 16]")
        if keys.dtype != _CODES or values.dtype != _CODES or not (keys.is_contiguous() and values.is_contiguous()):
            raise ValueError("cache codes must be contiguous E4M3 storage")
        scales = (layers, blocks, _KV_HEADS)
        for tensor in (key_scales, value_scales):
            if tensor.shape != scales or tensor.dtype is not _FLOAT or not tensor.is_contiguous():
                raise ValueError("cache scales must be contiguous FP32 [layers, blocks, 4]")
        _device(keys, values, key_scales, value_scales)

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


def _half(name: str, tensor: Tensor, index: int) -> None:
    if tensor.dtype is not _HALF or tensor.get_device() != index:
        raise ValueError(f"{name} must be FP16 on cuda:{index}")


def _int_list(index: int, name: str, tensor: Tensor, count: int) -> int:
    """Address of ``count`` or more int32 values on the device."""
    _fits(f"the entries of {name}", count)
    if tensor.dtype is _INT and tensor.numel() >= count and tensor.get_device() == index and tensor.is_contiguous():
        return tensor.data_ptr()
    raise ValueError(f"{name} must hold {count} contiguous int32 values on cuda:{index}")


def _check_rope(index: int, table: Tensor) -> int:
    if (
        table.dtype is _HALF
        and table.get_device() == index
        and table.shape == (2, 2048, 32)
        and table.is_contiguous()
    ):
        return table.data_ptr()
    raise ValueError(f"rope_table must be contiguous FP16 [2, 2048, 32] on cuda:{index}")


def _rows_ok(tensor: Tensor, strides: tuple[int, ...]) -> bool:
    """Inner [heads, 64] contiguous and rows 16-byte aligned."""
    return (
        strides[-1] == 1
        and strides[-2] == _HEAD_DIM
        and strides[0] % 8 == 0
        and strides[-3] % 8 == 0
        and tensor.data_ptr() % 16 == 0
    )


def _rows_apart(strides: tuple[int, ...], layers: int, tokens: int) -> bool:
    """Whether the [32, 64] rows of [layers, tokens, 32, 64] do not overlap: one of the two dimensions within the other."""
    over, within = strides[0], strides[1]
    if layers < 2 or tokens < 2:
        return (layers < 2 or over >= _ROW) and (tokens < 2 or within >= _ROW)
    if over < within:
        over, within, tokens = within, over, layers
    return within >= _ROW and over >= (tokens - 1) * within + _ROW


def _mixes(query: Tensor, out: Tensor) -> bool:
    """Whether a row of ``out`` may be written before another row of ``query`` that it overlaps is read.

    Both [layers, tokens, 32, 64] with contiguous rows, the query FP16; in place is fine.
    """
    layers, tokens = query.shape[0] - 1, query.shape[1] - 1
    first, strides = query.data_ptr(), query.stride()
    begin, over = out.data_ptr(), out.stride()
    if first == begin and strides == over and out.dtype is _HALF:
        return False
    last = first + 2 * (layers * strides[0] + tokens * strides[1] + _ROW)
    end = begin + out.element_size() * (layers * over[0] + tokens * over[1] + _ROW)
    return begin < last and first < end


def _dense(tensor: Tensor) -> Tensor:
    """A copy in contiguous, 16-byte aligned storage (``contiguous()`` keeps an unaligned tensor)."""
    return tensor.clone(memory_format=torch.contiguous_format)


def _aligned_pair(key: Tensor, value: Tensor) -> tuple[Tensor, Tensor, tuple[int, ...]]:
    """K and V with common strides that the kernels take (copies where they are not), and those strides."""
    strides = key.stride()
    if not (value.stride() == strides and _rows_ok(key, strides) and value.data_ptr() % 16 == 0):
        key, value = _dense(key), _dense(value)
        strides = key.stride()
    return key, value, strides


def _query_rows(query: Tensor) -> tuple[Tensor, int]:
    """Query [rows, 32, 64] as the kernels take it (a copy where it is not), and its row stride."""
    strides = query.stride()
    if strides[1:] == (_HEAD_DIM, 1) and query.data_ptr() % 16 == 0:
        if query.shape[0] == 1:
            return query, _ROW  # of one row the stride may be anything
        if strides[0] >= _ROW and strides[0] % 8 == 0:
            return query, strides[0]
    return _dense(query), _ROW


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
    [layers, tokens, 32, 64] is returned rotated: in FP32, unrounded, for
    ``prefill_attention``, or in ``query_out``, FP16 (which may be ``query``
    itself) or FP32.  The tokens of one block must be
    consecutive, in the list and in the block, as a request's positions are.
    """
    index = cache.key_codes.get_device()
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
    if layers == 0 or tokens == 0:
        return query_out
    key, value, strides = _aligned_pair(key, value)
    layer_stride, token_stride = strides[0], strides[1]
    _call(index, lib.pkv_fp8_append_kv, *cache._args(), layer_begin, layers, key.data_ptr(), value.data_ptr(),
          layer_stride, token_stride, slots_ptr, positions_ptr, tokens, rope, q_ptr, *q_strides, out_ptr,
          query_out is not None and query_out.dtype is _FLOAT, *out_strides,
          flag)
    return query_out


def read_blocks(cache: Fp8Cache, layer: int, blocks: Tensor, error_flag: Tensor) -> tuple[Tensor, Tensor]:
    """K and V of ``blocks`` (int32 [count]) at ``layer`` as FP16 [count, 16, 4, 64] each."""
    index = cache.key_codes.get_device()
    count = blocks.numel()
    blocks_ptr = _int_list(index, "blocks", blocks, count)
    flag = _int_list(index, "error_flag", error_flag, 1)
    key = torch.empty(count, _BLOCK_TOKENS, _KV_HEADS, _HEAD_DIM, dtype=_HALF, device=blocks.device)
    value = torch.empty_like(key)
    if count:
        _call(index, lib.pkv_fp8_read_blocks, *cache._args(), layer, blocks_ptr, count, key.data_ptr(),
              value.data_ptr(), flag)
    return key, value


_SAVED_BYTES = 2 * _KV_HEADS * (_BLOCK_TOKENS * _HEAD_DIM + 4)  # of a block in one layer


def save_blocks(cache: Fp8Cache, slots: Tensor) -> Tensor:
    """What ``restore_blocks`` needs to undo writes that begin at ``slots`` (int32 [count], one a block).

    A write inside a block may raise the block's scale and round its earlier
    codes again; this keeps the blocks' codes and scales, of every layer.
    """
    index = cache.key_codes.get_device()
    count = slots.numel()
    saved = torch.empty(max(count, 1) * cache.layers * _SAVED_BYTES, dtype=torch.uint8, device=cache.device)
    _call(index, lib.pkv_fp8_save_blocks, *cache._args(), _int_list(index, "slots", slots, count), count,
          saved.data_ptr(), saved.numel(), 0)
    return saved


def restore_blocks(cache: Fp8Cache, slots: Tensor, saved: Tensor) -> None:
    """The blocks of ``slots`` as they were when ``save_blocks`` returned ``saved``."""
    index = cache.key_codes.get_device()
    if saved.dtype is not torch.uint8 or saved.get_device() != index or not saved.is_contiguous():
        raise ValueError("saved must be what save_blocks returned")
    count = slots.numel()
    _call(index, lib.pkv_fp8_save_blocks, *cache._args(), _int_list(index, "slots", slots, count), count,
          saved.data_ptr(), saved.numel(), 1)


@functools.lru_cache(maxsize=4096)
def decode_plan(device_index: int, batch: int, total_blocks: int) -> tuple[int, int]:
    """Grid and workspace bytes of the decode attention (``pkv_fp8_decode_plan``)."""
    grid, workspace = ctypes.c_int32(), ctypes.c_int64()
    check(lib.pkv_fp8_decode_plan(device_index, batch, total_blocks, ctypes.byref(grid), ctypes.byref(workspace)))
    return grid.value, workspace.value


def decode_workspace_bytes(batch: int, grid: int) -> int:
    """Workspace of a decode launch with ``grid`` pieces (rotated queries, then split partials)."""
    return 2 * batch * _QUERY_HEADS * _HEAD_DIM * 2 + (batch + grid) * _QUERY_HEADS * (_HEAD_DIM + 2) * 4


def _attention_rows(name: str, tensor: Tensor, shape: tuple[int, ...], index: int) -> None:
    if tensor.shape != shape or tensor.dtype is not _HALF or tensor.get_device() != index:
        raise ValueError(f"{name} must be FP16 {list(shape)} on cuda:{index}")


def _query_and_out(
    query: Tensor, out: Tensor | None, index: int, rows: str, fp32: bool = False
) -> tuple[Tensor, int, Tensor, int]:
    """Query and output [rows, 32, 64] as the kernels take them, with their row strides."""
    shape = query.shape
    if len(shape) != 3 or shape[0] < 1 or shape[1] != _QUERY_HEADS or shape[2] != _HEAD_DIM:
        raise ValueError(f"query must be FP16 [{rows}, 32, 64] of a nonempty {rows}")
    if not (fp32 and query.dtype is _FLOAT and query.get_device() == index):
        _half("query", query, index)
    query, stride = _query_rows(query)
    if out is None:
        return query, stride, torch.empty_like(query, dtype=_HALF, memory_format=torch.contiguous_format), _ROW
    _attention_rows("out", out, shape, index)
    strides = out.stride()
    if not _rows_ok(out, strides):
        raise ValueError(f"out must be FP16 [{rows}, 32, 64] with contiguous, 16-byte aligned rows")
    return query, stride, out, _row_stride("out", out, _ROW)


def _decode(cache, layer, query, new, lengths, prefix, flat, total_blocks, error_flag, out) -> Tensor:
    index = cache.key_codes.get_device()
    query, query_stride, out, out_stride = _query_and_out(query, out, index, "batch")
    batch = query.shape[0]
    grid, workspace_bytes = decode_plan(index, batch, total_blocks)
    workspace = torch.empty((workspace_bytes + 1) // 2, dtype=_HALF, device=query.device)
    _call(
        index, lib.pkv_fp8_decode_attention if new is None else lib.pkv_fp8_decode_layer_zero, *cache._args(), layer,
        query.data_ptr(), query_stride, *(new or ()), _int_list(index, "lengths", lengths, batch),
        _int_list(index, "prefix", prefix, batch + 1), _int_list(index, "flat", flat, total_blocks), batch,
        total_blocks, grid, out.data_ptr(), out_stride, workspace.data_ptr(), workspace_bytes,
        _int_list(index, "error_flag", error_flag, 1),
    )
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
    return _decode(cache, layer, query, None, lengths, prefix, flat, total_blocks, error_flag, out)


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
    a last block.  A row without blocks gives zeros.
    """
    index = cache.key_codes.get_device()
    shape = (query.shape[0], _KV_HEADS, _HEAD_DIM)
    _attention_rows("key", key, shape, index)
    _attention_rows("value", value, shape, index)
    rope = _check_rope(index, rope_table)
    key, value, strides = _aligned_pair(key, value)
    new = (key.data_ptr(), value.data_ptr(), strides[0], rope)
    return _decode(cache, layer, query, new, lengths, prefix, flat, total_blocks, error_flag, out)


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
    """``kernels.prefill_attention`` over the 8-bit cache: rotated query [T, 32, 64], FP16 or FP32.

    Token t attends to positions 0 .. start + t through ``blocks`` (int32, the
    request's physical block per 16 positions).  A V value that is NaN may also
    reach tokens up to 63 positions before it (their weight for it is 0).
    """
    index = cache.key_codes.get_device()
    query, query_stride, out, out_stride = _query_and_out(query, out, index, "tokens", fp32=True)
    tokens = query.shape[0]
    if type(start) is not int or start < 0 or start + tokens > 2048:
        raise ValueError("the chunk must hold 1 or more tokens at positions below 2048")
    count = -(-(start + tokens) // _BLOCK_TOKENS)
    blocks_ptr = _int_list(index, "blocks", blocks, count)
    workspace = torch.empty(count * _PREFILL_BLOCK_BYTES // 2, dtype=_HALF, device=out.device)
    _call(index, lib.pkv_fp8_prefill_attention, *cache._args(), layer, query.data_ptr(), query.dtype is _FLOAT,
          query_stride, blocks_ptr, start, tokens, out.data_ptr(), out_stride, workspace.data_ptr(),
          count * _PREFILL_BLOCK_BYTES, _int_list(index, "error_flag", error_flag, 1))
    return out
