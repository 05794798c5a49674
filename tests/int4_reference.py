"""64-bit restatement of the 4-bit KV cache, for its tests (plain torch, any device)."""

from __future__ import annotations

import math

import torch

from pagedcore_b200 import int4, rope

# The number that each scale byte stands for: 5 exponent and 3 fraction bits, no sign.
NUMBERS = [math.ldexp(b % 8 + 8 * (b > 7), max(b // 8, 1) - 18) for b in range(248)]
LARGEST = 9216.0
LAYERS, LAYER = 3, 1


def numbers(device) -> torch.Tensor:
    return torch.tensor([n for n in NUMBERS if n <= LARGEST], dtype=torch.float64, device=device)


def scale_for(amax: torch.Tensor) -> torch.Tensor:
    """The scale of groups with the largest magnitude ``amax``: nearest to a seventh, even byte at ties."""
    known = numbers(amax.device)
    want = amax.double()[..., None]
    off = (7 * known - want).abs()
    byte = torch.arange(len(known), device=amax.device)
    nearest = torch.where(off == off.amin(-1, keepdim=True), byte % 2, 2).argmin(-1)
    up = (7 * known < want).sum(-1).clamp(max=len(known) - 1)
    return known[torch.where(amax.double() < 7 * 2.0**-14, up, nearest)]


def stored(values: torch.Tensor) -> torch.Tensor:
    """What the cache holds for FP32 ``values`` [..., 64]: float64, NaN in groups that are not finite."""
    groups = values.double().unflatten(-1, (4, 16))
    finite = groups.isfinite().all(-1, keepdim=True)
    groups = torch.where(finite, groups, 0.0)
    scale = scale_for(groups.abs().amax(-1))[..., None]
    codes = torch.round(groups / torch.where(scale > 0, scale, 1.0)).clamp(-7, 7)
    return torch.where(finite, codes * scale, math.nan).flatten(-2)


def rope64(rows: torch.Tensor, table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """[tokens, heads, 64] rotated at int64 positions, in float64."""
    cos, sin = (t[positions].double()[:, None] for t in table)
    low, high = rows[..., :32].double(), rows[..., 32:].double()
    return torch.cat((low * cos - high * sin, high * cos + low * sin), -1)


def norm64(rows: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    x = rows.double()
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def unpack(storage: torch.Tensor, block: int, head: int, token: int) -> tuple[list[int], list[int], list[int], list[int]]:
    """K codes, K scale bytes, V codes and V scale bytes of one token and head of a layer [blocks, 4608]."""
    raw = storage[block, 1152 * head : 1152 * (head + 1)].tolist()

    def codes(word: list[int]) -> list[int]:
        out = [0] * 8
        for h in (0, 1):
            half = word[2 * h] | word[2 * h + 1] << 8
            half = (half >> 2 | half << 14) & 0xFFFF
            for i in range(4):
                out[2 * i + h] = (half >> 4 * i & 15) - 8
        return out

    key, value = [], []
    for chunk in range(8):
        at = chunk // 2 * 128 + token * 8 + chunk % 2 * 4
        key += codes(raw[at : at + 4])
        at = 512 + chunk * 64 + token * 4
        value += codes(raw[at : at + 4])
    return (key, [raw[1024 + 16 * t + token] for t in range(4)], value, [raw[1088 + 16 * t + token] for t in range(4)])


class Case:
    """A cache of garbage with rows of given lengths written into scattered blocks, and what it then holds."""

    def __init__(self, seed: int, lengths: list[int], spare: int = 3, spread: float = 0.0, device="cuda") -> None:
        generator = torch.Generator().manual_seed(seed)
        counts = [-(-n // 16) for n in lengths]
        blocks = sum(counts) + spare
        self.device = torch.device(device)
        storage = torch.randint(0, 256, (LAYERS, blocks, int4.BLOCK_BYTES), dtype=torch.uint8, generator=generator)
        storage.view(LAYERS, blocks, 4, 1152)[..., 1024:] = 255  # scales that are NaN wherever nothing is written
        self.cache = int4.Int4Cache(storage.to(self.device))
        self.flag = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.rope = rope.device_table(self.device)
        order = torch.randperm(blocks, generator=generator).tolist()
        self.tables = [[order.pop() for _ in range(count)] for count in counts]
        self.free, self.lengths = order, list(lengths)
        self.held = {name: torch.full((blocks, 16, 4, 64), math.nan, dtype=torch.float64, device=self.device)
                     for name in ("key", "value")}
        for row, length in enumerate(lengths):
            if length:
                draw = lambda: torch.randn(length, 4, 64, generator=generator).to(self.device)  # noqa: E731
                factor = torch.exp2(spread * torch.randn(length, 1, 1, generator=generator)).to(self.device)
                self.append(row, draw() * factor, draw() * factor, 0)

    def slots(self, row: int, start: int, count: int) -> torch.Tensor:
        at = [self.tables[row][p // 16] * 16 + p % 16 for p in range(start, start + count)]
        return torch.tensor(at, dtype=torch.int32, device=self.device)

    def hold(self, slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> None:
        """FP32 rows [tokens, 4, 64] were written at ``slots``."""
        block, slot = slots.long() // 16, slots.long() % 16
        self.held["key"][block, slot], self.held["value"][block, slot] = stored(key), stored(value)

    def append(self, row: int, key: torch.Tensor, value: torch.Tensor, start: int) -> None:
        slots = self.slots(row, start, key.shape[0])
        int4.append_kv(self.cache, key.half()[None], value.half()[None], slots, layer_begin=LAYER, error_flag=self.flag)
        self.hold(slots, key.half().float(), value.half().float())

    def batch(self):
        """lengths, prefix, flat on the device and the block count."""
        flat = [block for table in self.tables for block in table]
        prefix = [0]
        for table in self.tables:
            prefix.append(prefix[-1] + len(table))
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
        return as_int(self.lengths), as_int(prefix), as_int(flat), len(flat)

    def tokens(self, row: int, length: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V [length, 4, 64] of a row, in float64."""
        length = self.lengths[row] if length is None else length
        return tuple(self.held[name][self.tables[row]].reshape(-1, 4, 64)[:length] for name in ("key", "value"))

    def check_values(self) -> None:
        """What the cache holds at every written slot, to the bit."""
        for row, length in enumerate(self.lengths):
            if length:
                blocks = torch.tensor(self.tables[row], dtype=torch.int32, device=self.device)
                for got, want in zip(int4.read_blocks(self.cache, LAYER, blocks, self.flag), self.tokens(row)):
                    got = got.reshape(-1, 4, 64)[:length].double()
                    assert torch.equal(got.nan_to_num(9e9), want.nan_to_num(9e9)), row
        assert int(self.flag.item()) == 0
