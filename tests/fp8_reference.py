"""64-bit restatement of the 8-bit operators, for their tests (plain torch, any device)."""

from __future__ import annotations

import math

import torch

HALF_E4M3 = 2.0**-4  # half a step of E4M3, relative to a normal value
HALF_FP16 = 2.0**-11
F32 = 2.0**-24


def scale_for(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two in [2^-15, 2^8] with amax / scale <= 448 (float64)."""
    exponents = torch.arange(-15, 9, dtype=torch.int32, device=amax.device)
    powers = torch.ldexp(torch.ones(24, dtype=torch.float64, device=amax.device), exponents)
    return powers[(amax.double()[..., None] > 448 * powers).sum(-1).clamp(max=23)]


def finite_amax(values: torch.Tensor, dims) -> torch.Tensor:
    return torch.where(values.isfinite(), values.abs(), 0.0).amax(dims)


def round_e4m3(values: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The value that E4M3 with ``scale`` stores for each of ``values``; not finite -> NaN."""
    v = values.double() / scale
    exponent = torch.frexp(v.abs().clamp(min=2.0**-6))[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    limit = torch.where(scale == 256.0, 240.0, 448.0).double()
    rounded = torch.minimum(torch.maximum(torch.round(v / step) * step, -limit), limit) * scale
    return torch.where(values.isfinite(), rounded, math.nan)


def group_amax(values: torch.Tensor) -> torch.Tensor:
    """[rows, width] -> [rows, ceil(width / 128)] largest finite magnitudes."""
    rows, width = values.shape
    groups = -(-width // 128)
    padded = torch.nn.functional.pad(values, (0, 128 * groups - width))
    return finite_amax(padded.view(rows, groups, 128), -1)


def spread(scales: torch.Tensor, width: int) -> torch.Tensor:
    return scales.double().repeat_interleave(128, 1)[:, :width]


def check_rows(actual, exact: torch.Tensor, relative: float) -> None:
    """``actual`` (Fp8Rows) holds ``exact`` rounded once, computed with a relative error of ``relative``.

    A scale may be that of an amax off by the error; a value is off by half a
    step of E4M3 (2^-4 of it, or half the subnormal step, 2^-10 of the scale)
    on top of the error.
    """
    codes, scales = actual.codes, actual.scales
    amax = group_amax(exact)
    low, high = scale_for(amax * (1 - relative)), scale_for(amax * (1 + relative))
    assert bool(((scales.double() == low) | (scales.double() == high)).all())
    values = codes.double() * spread(scales, exact.shape[1])
    bad = ~exact.isfinite()
    assert torch.equal(values.isnan(), bad)
    step = torch.maximum(HALF_E4M3 * exact.abs(), spread(scales, exact.shape[1]) * 2.0**-10)
    bound = step * (1 + relative) + relative * exact.abs()
    assert bool(((values - exact).abs() <= bound)[~bad].all())


def rope64(rows: torch.Tensor, table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """[tokens, heads, 64] rotated at int64 positions."""
    cos, sin = (t[positions].double()[:, None] for t in table)
    low, high = rows[..., :32].double(), rows[..., 32:].double()
    return torch.cat((low * cos - high * sin, high * cos + low * sin), -1)


class CacheOracle:
    """The values of one layer's K or V: float64 [blocks, 4, 16, 64] and the scale of each tile."""

    def __init__(self, blocks: int, device) -> None:
        self.values = torch.zeros(blocks, 4, 16, 64, dtype=torch.float64, device=device)
        self.scale = torch.full((blocks, 4), 2.0**-15, dtype=torch.float64, device=device)

    def append(self, rows: torch.Tensor, slots: list[int]) -> None:
        """rows [tokens, 4, 64] at slots, block by block in order."""
        at = 0
        while at < len(slots):
            block, first = divmod(slots[at], 16)
            run = 1
            while at + run < len(slots) and slots[at + run] == slots[at] + run and first + run < 16:
                run += 1
            new = rows[at : at + run].double().transpose(0, 1)  # [4, run, 64]
            scale = scale_for(finite_amax(new, (1, 2)))
            if first:
                scale = torch.maximum(scale, self.scale[block])
            self.scale[block] = scale
            self.values[block, :, :first] = round_e4m3(self.values[block, :, :first], scale[:, None, None])
            self.values[block, :, first : first + run] = round_e4m3(new, scale[:, None, None])
            at += run

    def tokens(self, table: list[int], length: int) -> torch.Tensor:
        """[length, 4, 64] of a block table."""
        return self.values[table].transpose(1, 2).reshape(-1, 4, 64)[:length]


def attend64(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, weight_error: float = 2.0**-21):
    """One query [32, 64] over K/V [tokens, 4, 64] (float64): output [32, 64] and its error bound.

    A softmax weight is off by ``weight_error`` as the second product takes it
    (2^-22 and the rounding of its low half in the decode kernels, 2^-11 in the
    prompt kernel), and by the error of its score: 64 exact products summed in
    FP32 (65 roundings of the summed magnitudes, 2^-24 each, twice over for two
    halves of a query, and as much again for truncation inside the tensor
    core; the scale, the subtraction of the maximum and 2^x add 2^-20 and two
    roundings of the score).  The second product sums in FP32 likewise, and the
    output is rounded to FP16.
    """
    if key.shape[0] == 0:
        zero = torch.zeros(32, 64, dtype=torch.float64, device=query.device)
        return zero, zero
    q = query.double().view(4, 8, 64)
    k, v = key.transpose(0, 1), value.transpose(0, 1)  # [4, tokens, 64]
    scores = q @ k.transpose(1, 2) / 8
    weights = torch.softmax(scores, -1)
    out = weights @ v
    magnitude = (q.abs() @ k.abs().transpose(1, 2) / 8).amax(-1, keepdim=True)
    off = 4 * 65 * F32 * magnitude + 2.0**-20 + 4 * F32 * scores.abs().amax(-1, keepdim=True)
    off = off + 2 * key.shape[0] * F32  # the sums over tokens
    bound = HALF_FP16 * out.abs() + (weight_error + 2 * off) * (weights @ v.abs()) + 2.0**-25
    return out.reshape(32, 64), bound.reshape(32, 64)
