"""What the 4-bit KV cache costs: cases, inputs, plain forms and 64-bit results.

Four operators, each as a user's program calls it:

- ``write``   new K (rotated, with or without a norm of each head first) and V of a list of
  tokens written into the cache, and the blocks that they went to read back as FP16.
- ``attend``  attention of one token a row over block tables, queries already rotated.
- ``decode``  one decode layer: the new token of each row written (norm and rotation of its
  query and K in the same pass), then the attention; the rows' last blocks read back.
- ``prompt``  one layer of a prompt chunk: queries rotated, K and V written, causal attention
  through the block table, the written blocks read back.

A group is 16 consecutive dims of one token and head.  It is stored as 16 codes of 4 bits
and one scale s of 8 bits: an unsigned number with 5 exponent and 3 fraction bits, the FP16
number whose bits 14 .. 7 it is.  s is the number nearest to a seventh of the group's largest
magnitude (below 2^-14 the next multiple of 2^-17 up, at most 9216), a code is x / s rounded to
nearest even, between -7 and 7, and a value is code times s.

The cache is bytes [layers, blocks, 4608], a block holding 16 tokens: for each of the 4 heads
512 bytes of K codes [4 groups][16 tokens][8 bytes], 512 of V codes [8 chunks][16 tokens][4 bytes]
(a chunk is 8 dims), 64 of K scales [4 groups][16 tokens] and 64 of V scales.  Eight codes lie in
four bytes as two 16-bit halves, dim 2 i + h being nibble i of half h; a half is stored rotated left
by two bits, and nibbles hold code + 8.
"""

from __future__ import annotations

import math

import torch

own = False

LAYERS, LAYER = 2, 1  # the cache holds two layers; single-layer calls use the second
KV_HEADS, GROUP, HEAD_DIM, BLOCK = 4, 8, 64, 16
QUERY_HEADS = KV_HEADS * GROUP
HEAD_BYTES = 1152  # of one head of a block
CONTEXT = 2048  # positions of the rotation table
MOST_TOKENS = 262144  # of an attention, over all rows
LARGEST = 225  # the scale 9216
EPS = 1e-5


def listed() -> list[dict]:
    return [
        # One sequence's new token in one layer: bound by launch latency.
        {"name": "write_token", "op": "write", "layers": 1, "tokens": 1, "apart": True, "norm": True},
        # The new tokens of this repository's benchmark batch (256 sequences), each in a block of its own.
        {"name": "write_batch", "op": "write", "layers": 1, "tokens": 256, "apart": True, "norm": True},
        # A finished prompt's K and V of several layers at once, as the allocator's append writes them.
        {"name": "write_prompt", "op": "write", "layers": 2, "tokens": 2047, "apart": False, "norm": False},
        # A short question behind a system prompt: one sequence, three blocks.
        {"name": "attend_short", "op": "attend", "batch": 1, "low": 41, "high": 41},
        # Two long documents: the long axis has to be split.
        {"name": "attend_long", "op": "attend", "batch": 2, "low": 131071, "high": 131072},
        # A ragged batch of conversations.
        {"name": "attend_batch", "op": "attend", "batch": 64, "low": 1, "high": 8190},
        # One short sequence: a partial block and its first neighbour.
        {"name": "decode_one", "op": "decode", "batch": 1, "low": 17, "high": 17, "norm": False},
        # A small batch of a model with head norms.
        {"name": "decode_few_norm", "op": "decode", "batch": 7, "low": 900, "high": 2048, "norm": True},
        # The benchmark's ragged batch: 256 sequences of 1 to 2048 tokens.
        {"name": "decode_batch", "op": "decode", "batch": 256, "low": 1, "high": 2048, "norm": False},
        # A short prompt continuing a cached conversation inside a block, with head norms.
        {"name": "prompt_continued", "op": "prompt", "start": 601, "tokens": 75, "norm": True},
        # A full-length prompt.
        {"name": "prompt_full", "op": "prompt", "start": 0, "tokens": 2047, "norm": False},
    ]


def _log(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    op = rng.choice(("write", "attend", "decode", "prompt"))
    norm = rng.random() < 0.5
    if op == "write":
        tokens = _log(rng, 1, 2047)
        apart = tokens <= 256 and rng.random() < 0.5
        return {"op": op, "layers": rng.randint(1, LAYERS), "tokens": tokens, "apart": apart, "norm": norm}
    if op == "attend":
        batch = _log(rng, 1, 64)
        high = _log(rng, 1, min(131072, MOST_TOKENS // batch))
        return {"op": op, "batch": batch, "low": rng.randint(1, high), "high": high}
    if op == "decode":
        high = _log(rng, 1, CONTEXT)
        return {"op": op, "batch": _log(rng, 1, 128), "low": rng.randint(1, high), "high": high, "norm": norm}
    tokens = _log(rng, 1, 1500)
    return {"op": op, "start": rng.randint(0, 2047 - tokens), "tokens": tokens, "norm": norm}


# -- numbers and storage -----------------------------------------------------------
def _scale_bytes(amax: torch.Tensor) -> torch.Tensor:
    """Scales (int32 0 .. 255) of groups with the largest magnitude ``amax`` (float32, finite)."""
    seventh = amax / torch.full_like(amax, 7)  # by the number 7 itself it would be a product with 1 / 7, not exact at ties
    bits = seventh.view(torch.int32)
    rounded = (bits + 0x7FFFF + ((bits >> 20) & 1) >> 20) - (112 << 3)
    small = torch.ceil(seventh * 2.0**17).int()
    return torch.where(seventh < 2.0**-14, small, rounded.clamp(max=LARGEST))


def _scale_values(scales: torch.Tensor) -> torch.Tensor:
    """The numbers that scale bytes stand for, in float32."""
    return (scales.int() << 7).short().view(torch.float16).float()


def _quantize(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 [..., 64] -> codes int32 [..., 64] in -7 .. 7 and scale bytes int32 [..., 4]."""
    groups = rows.unflatten(-1, (4, 16))
    scales = _scale_bytes(groups.abs().amax(-1))
    value = _scale_values(scales)[..., None]
    codes = torch.round(groups / torch.where(value > 0, value, 1.0)).clamp(-7, 7).int()
    return codes.flatten(-2), scales


def _pack(codes: torch.Tensor) -> torch.Tensor:
    """codes [..., 64] -> bytes [..., 32], four for each eight dims."""
    nibbles = (codes + 8).unflatten(-1, (8, 4, 2))  # chunk, nibble, half
    half = nibbles[..., 0, :] | nibbles[..., 1, :] << 4 | nibbles[..., 2, :] << 8 | nibbles[..., 3, :] << 12
    half = (half << 2 | half >> 14) & 0xFFFF
    return torch.stack((half & 0xFF, half >> 8), -1).flatten(-3).to(torch.uint8)


def _unpack(stored: torch.Tensor) -> torch.Tensor:
    """bytes [..., 32] -> float32 codes [..., 64]."""
    pairs = stored.int().unflatten(-1, (8, 2, 2))  # chunk, half, byte
    half = pairs[..., 0] | pairs[..., 1] << 8
    half = (half >> 2 | half << 14) & 0xFFFF
    nibbles = torch.stack([half >> 4 * i & 15 for i in range(4)], -2)  # [..., chunk, nibble, half]
    return (nibbles - 8).float().flatten(-3)


def _parts(layer: torch.Tensor, name: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of K or V in one layer's blocks, as views [blocks, heads, ..., tokens, ...]."""
    heads = layer.view(layer.shape[0], KV_HEADS, HEAD_BYTES)
    if name == "key":
        return heads[..., :512].unflatten(-1, (4, BLOCK, 8)), heads[..., 1024:1088].unflatten(-1, (4, BLOCK))
    return heads[..., 512:1024].unflatten(-1, (8, BLOCK, 4)), heads[..., 1088:].unflatten(-1, (4, BLOCK))


def _put(layer: torch.Tensor, name: str, block: torch.Tensor, slot: torch.Tensor, rows: torch.Tensor) -> None:
    """Write float32 ``rows`` [n, heads, 64] into ``slot`` [n] of ``block`` [n]."""
    stored_codes, stored_scales = _parts(layer, name)
    codes, scales = _quantize(rows)
    width = stored_codes.shape[-1]
    stored_codes[block, :, :, slot] = _pack(codes).unflatten(-1, (32 // width, width))
    stored_scales[block, :, :, slot] = scales.to(torch.uint8)


def _get(layer: torch.Tensor, name: str, blocks: torch.Tensor) -> torch.Tensor:
    """float32 values [n, 16, heads, 64] of ``blocks`` [n]."""
    codes, scales = (part[blocks] for part in _parts(layer, name))
    values = _unpack(codes.transpose(2, 3).flatten(-2))  # [n, heads, 16, 64]
    step = _scale_values(scales).transpose(-1, -2)[..., None]  # [n, heads, 16, 4, 1]
    return (values.unflatten(-1, (4, 16)) * step).flatten(-2).transpose(1, 2)


# -- inputs ------------------------------------------------------------------------
def _rope_table(device) -> torch.Tensor:
    """FP16 cos and sin [2, 2048, 32]."""
    inverse = 1.0 / (10000.0 ** (torch.arange(0, HEAD_DIM, 2).float() / HEAD_DIM))
    angles = torch.arange(CONTEXT).float()[:, None] * inverse
    return torch.stack((angles.cos(), angles.sin())).half().to(device)


def _history(generator, blocks: int, layers: int, device) -> torch.Tensor:
    """A filled cache [2, blocks, 4608]; the first layer is left zero when ``layers`` is 1."""
    storage = torch.zeros((LAYERS, blocks, KV_HEADS * HEAD_BYTES), dtype=torch.uint8, device=device)
    channels = 0.5 + 2.5 * torch.rand((HEAD_DIM,), device=device, generator=generator) ** 4  # a few strong K channels
    for layer in range(LAYERS - layers, LAYERS):
        for name, spread in (("key", channels), ("value", 1.0)):
            for at in range(0, blocks, 4096):
                count = min(4096, blocks - at)
                rows = torch.randn((count, BLOCK, KV_HEADS, HEAD_DIM), device=device, generator=generator) * spread
                codes, scales = _quantize(rows)  # every token of the block at once
                stored_codes, stored_scales = _parts(storage[layer, at : at + count], name)
                width = stored_codes.shape[-1]
                stored_codes.copy_(_pack(codes).unflatten(-1, (32 // width, width)).permute(0, 2, 3, 1, 4))
                stored_scales.copy_(scales.permute(0, 2, 3, 1))
    return storage


def _clear(storage: torch.Tensor, block: torch.Tensor, used: torch.Tensor) -> None:
    """Zero the never-written slots (``used`` and later) of ``block`` in every layer."""
    keep = torch.arange(BLOCK, device=block.device) < used[:, None]  # [blocks, 16]
    for layer in storage:
        for name in ("key", "value"):
            codes, scales = _parts(layer, name)
            codes[block] = codes[block] * keep[:, None, None, :, None]
            scales[block] = scales[block] * keep[:, None, None, :]


def _lengths(case: dict) -> list[int]:
    batch, low, high = case["batch"], case["low"], case["high"]
    return [low + (high - low) * i // max(1, batch - 1) for i in range(batch)]


def prepare(case: dict, seed: int) -> dict:
    device = torch.device("cuda")
    generator = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=device, generator=generator)

    def order(count):
        return torch.randperm(count, device=device, generator=generator)

    op = case["op"]
    state = {"case": case, "rope": _rope_table(device)}
    state["error_flag"] = torch.zeros(1, dtype=torch.int32, device=device)
    layers = 1
    if op in ("attend", "decode"):
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=device)[order(case["batch"])]
        counts = (lengths + BLOCK - 1) // BLOCK
        prefix = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).int()
        rows = case["batch"]
        total = sum(-(-n // BLOCK) for n in _lengths(case))
        storage = _history(generator, total + 3, 1, device)
        flat = order(total + 3)[:total].int()
        last = flat[(prefix[1:] - 1).long()]
        state |= {"lengths": lengths, "prefix": prefix, "total_blocks": total, "last": last}
        _clear(storage, last.long(), (lengths.long() - 1) % BLOCK + (op == "attend"))
    elif op == "prompt" or not case["apart"]:
        start, rows = case.get("start", 0), case["tokens"]
        total = -(-(start + rows) // BLOCK)
        layers = case.get("layers", 1)
        storage = _history(generator, total + 3, layers, device)
        flat = order(total + 3)[:total].int()
        positions = torch.arange(start, start + rows, dtype=torch.int32, device=device)
        state["slots"] = flat[positions.long() // BLOCK] * BLOCK + positions % BLOCK
        state["written"] = flat[start // BLOCK :].contiguous()
        state["positions"] = positions
        used = (start - BLOCK * torch.arange(start // BLOCK, total, device=device)).clamp(0, BLOCK)
        _clear(storage, state["written"].long(), used)
    else:
        rows, layers = case["tokens"], case["layers"]
        storage = _history(generator, rows + 3, layers, device)
        flat = order(rows + 3)[:rows].int()
        positions = torch.randint(0, CONTEXT, (rows,), device=device, generator=generator, dtype=torch.int32)
        state["slots"] = flat * BLOCK + positions % BLOCK
        state["written"] = flat
        state["positions"] = positions
        _clear(storage, flat.long(), positions.long() % BLOCK)
    state |= {"storage": storage, "flat": flat}
    if op != "write":
        state["query"] = normal(rows, QUERY_HEADS, HEAD_DIM).half()
    if op != "attend":
        state["key"] = (normal(layers, rows, KV_HEADS, HEAD_DIM) * 1.2).half()
        state["value"] = normal(layers, rows, KV_HEADS, HEAD_DIM).half()
        if case["norm"]:
            state["query_norm"], state["key_norm"] = ((1 + 0.1 * normal(LAYERS, HEAD_DIM)).half() for _ in range(2))
    return state


# -- plain forms ---------------------------------------------------------------------
def _rotated(rows: torch.Tensor, norm: torch.Tensor | None, state: dict, positions: torch.Tensor) -> torch.Tensor:
    """Norm of each head (where there is one) and RoPE of [tokens, heads, 64] at int64 positions.

    In 64 bits and rounded to 32 once: K is rounded to codes next, and a value beside the border
    between two of them must not depend on the order of a sum.
    """
    x = rows.double()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.double()
    cos, sin = (table[positions].double().repeat(1, 2)[:, None] for table in state["rope"])
    return (x * cos + torch.cat((-x[..., 32:], x[..., :32]), -1) * sin).float()


def _softmax(scores: torch.Tensor) -> torch.Tensor:
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return weights / weights.sum(-1, keepdim=True)


def _write_layers(state: dict, layer_begin: int, positions: torch.Tensor, slots: torch.Tensor) -> None:
    block, slot = slots // BLOCK, slots % BLOCK
    for index in range(state["key"].shape[0]):
        norm = state["key_norm"][layer_begin + index] if state["case"]["norm"] else None
        layer = state["storage"][layer_begin + index]
        _put(layer, "key", block, slot, _rotated(state["key"][index], norm, state, positions))
        _put(layer, "value", block, slot, state["value"][index].float())


def _read(state: dict, layer: int, blocks: torch.Tensor):
    """K and V [blocks, 16, heads, 64] FP16."""
    return tuple(_get(state["storage"][layer], name, blocks.long()).half() for name in ("key", "value"))


def _write(state: dict):
    begin = LAYERS - state["case"]["layers"]
    _write_layers(state, begin, state["positions"].long(), state["slots"].long())
    return [_read(state, layer, state["written"]) for layer in range(begin, LAYERS)]


def _attend_rows(state: dict, query: torch.Tensor) -> torch.Tensor:
    lengths, prefix = state["lengths"].long(), state["prefix"].long()
    batch, most = lengths.shape[0], -(-state["case"]["high"] // BLOCK)
    at = (prefix[:-1, None] + torch.arange(most, device=prefix.device)).clamp(max=state["total_blocks"] - 1)

    def rows(name):
        values = _get(state["storage"][LAYER], name, state["flat"].long())
        return values[at].reshape(batch, most * BLOCK, KV_HEADS, HEAD_DIM).transpose(1, 2)

    scores = query.view(batch, KV_HEADS, GROUP, HEAD_DIM) @ rows("key").transpose(-1, -2) * HEAD_DIM**-0.5
    beyond = (torch.arange(most * BLOCK, device=lengths.device) >= lengths[:, None])[:, None, None]
    weights = _softmax(scores.masked_fill(beyond, -math.inf))
    values = rows("value").masked_fill(beyond.transpose(-1, -2), 0.0)
    return (weights @ values).view(batch, QUERY_HEADS, HEAD_DIM).half()


def _attend(state: dict):
    return _attend_rows(state, state["query"].float())


def _decode(state: dict):
    positions, last = state["lengths"].long() - 1, state["last"].long()
    _write_layers(state, LAYER, positions, last * BLOCK + positions % BLOCK)
    norm = state["query_norm"][LAYER] if state["case"]["norm"] else None
    out = _attend_rows(state, _rotated(state["query"], norm, state, positions))
    return out, _read(state, LAYER, last)


def _prompt(state: dict):
    tokens, positions = state["case"]["tokens"], state["positions"].long()
    total = state["case"]["start"] + tokens
    norm = state["query_norm"][LAYER] if state["case"]["norm"] else None
    query = _rotated(state["query"], norm, state, positions)
    _write_layers(state, LAYER, positions, state["slots"].long())
    keys, values = (
        _get(state["storage"][LAYER], name, state["flat"].long()).flatten(0, 1)[:total].transpose(0, 1)
        for name in ("key", "value")
    )  # [heads, total, 64]
    grouped = query.view(tokens, KV_HEADS, GROUP, HEAD_DIM).permute(1, 2, 0, 3)
    scores = grouped @ keys[:, None].transpose(-1, -2) * HEAD_DIM**-0.5
    beyond = torch.arange(total, device=positions.device) > positions[:, None]
    out = _softmax(scores.masked_fill(beyond, -math.inf)) @ values[:, None]
    return out.permute(2, 0, 1, 3).reshape(tokens, QUERY_HEADS, HEAD_DIM).half(), _read(state, LAYER, state["written"])


def _run_own(state: dict):
    from pagedcore_b200 import int4

    op, flag = state["case"]["op"], state["error_flag"]
    cache = int4.Int4Cache(state["storage"])
    if op == "attend":
        return int4.decode_attention(
            cache, LAYER, state["query"], state["lengths"], state["prefix"], state["flat"], state["total_blocks"], flag
        )
    norms = int4.HeadNorms(state["query_norm"], state["key_norm"], EPS) if state["case"]["norm"] else None
    if op == "decode":
        out = int4.decode_layer(
            cache, LAYER, state["query"], state["key"][0], state["value"][0], state["rope"], state["lengths"],
            state["prefix"], state["flat"], state["total_blocks"], flag, norms=norms,
        )
        return out, int4.read_blocks(cache, LAYER, state["last"], flag)
    begin = LAYERS - state["key"].shape[0]
    query = int4.append_kv(
        cache, state["key"], state["value"], state["slots"], layer_begin=begin, error_flag=flag,
        positions=state["positions"], rope_table=state["rope"],
        query=state["query"][None] if op == "prompt" else None, norms=norms,
    )
    if op == "write":
        return [int4.read_blocks(cache, layer, state["written"], flag) for layer in range(begin, LAYERS)]
    out = int4.prefill_attention(cache, LAYER, query[0], state["flat"], state["case"]["start"], flag)
    return out, int4.read_blocks(cache, LAYER, state["written"], flag)


_PLAIN = {"write": _write, "attend": _attend, "decode": _decode, "prompt": _prompt}


def run(state: dict):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# -- what a pass cannot do without --------------------------------------------------------
def work(case: dict) -> dict:
    op = case["op"]
    token = 2 * KV_HEADS * (HEAD_DIM // 2 + HEAD_DIM // 16)  # bytes of one token in the cache
    fresh = 2 * KV_HEADS * HEAD_DIM * 2  # of its K and V in FP16
    head = QUERY_HEADS * HEAD_DIM * 2  # of a row's queries, or of its output
    if op == "write":
        blocks = case["tokens"] if case["apart"] else -(-case["tokens"] // BLOCK)
        one = case["tokens"] * (fresh + token) + blocks * BLOCK * (token + fresh)
        return {"bytes": case["layers"] * one, "flops": case["layers"] * case["tokens"] * 2 * KV_HEADS * HEAD_DIM * 6}
    if op == "prompt":
        start, rows = case["start"], case["tokens"]
        tokens, pairs = start + rows, rows * start + rows * (rows + 1) // 2
        back = -(-tokens // BLOCK) - start // BLOCK
    else:
        tokens = pairs = sum(_lengths(case))
        rows = back = case["batch"]
    moved = tokens * token + 2 * rows * head
    if op != "attend":
        moved += rows * (fresh + token) + back * BLOCK * (token + fresh)
    return {"bytes": moved, "flops": 4 * pairs * QUERY_HEADS * HEAD_DIM}


# -- the same in 64 bits -------------------------------------------------------------------
def _numbers(device) -> torch.Tensor:
    """The 256 scales' numbers in float64: exponent 0 counts in steps of 2^-17."""
    numbers = [math.ldexp(byte % 8 + 8 * (byte > 7), max(byte // 8, 1) - 18) for byte in range(256)]
    return torch.tensor(numbers, dtype=torch.float64, device=device)


def _exact_rounded(rows: torch.Tensor) -> torch.Tensor:
    """float64 [..., 64] -> the values that the cache holds for them."""
    numbers = _numbers(rows.device)[: LARGEST + 1]
    out = torch.empty_like(rows)
    for at in range(0, HEAD_DIM, 16):
        part = rows[..., at : at + 16]
        want = part.abs().amax(-1, keepdim=True)  # 7 scales, nothing divided
        above = torch.searchsorted(7 * numbers, want.contiguous()).clamp(max=LARGEST)  # the first not below it
        below = (above - 1).clamp(min=0)
        up, down = 7 * numbers[above] - want, want - 7 * numbers[below]
        lower = (down < up) | ((down == up) & (below % 2 == 0))
        scale = numbers[torch.where((want >= 7 * 2.0**-14) & lower & (up >= 0), below, above)]
        code = torch.round(part / torch.where(scale > 0, scale, 1.0))
        out[..., at : at + 16] = code.clamp(-7, 7) * scale
    return out


def _exact_stored(state: dict, layer: int, blocks: torch.Tensor):
    """K and V [n, 16, heads, 64] in float64, taken from the stored bytes."""
    raw = state["storage"][layer][blocks].view(-1, KV_HEADS, HEAD_BYTES).long()
    numbers = _numbers(raw.device)
    found = []
    for name in ("key", "value"):
        at, unit = (0, 8) if name == "key" else (512, 4)  # first byte, bytes of a token's run
        out = torch.empty((raw.shape[0], BLOCK, KV_HEADS, HEAD_DIM), dtype=torch.float64, device=raw.device)
        scales = numbers[raw[..., 1024 if name == "key" else 1088 :][..., :64]].view(-1, KV_HEADS, 4, BLOCK)
        for dim in range(HEAD_DIM):
            byte = dim // 8 * 4  # of the token's 32, where its chunk begins
            first = at + byte // unit * BLOCK * unit + byte % unit + 2 * (dim % 2)
            places = first + unit * torch.arange(BLOCK, device=raw.device)
            half = raw[..., places] + 256 * raw[..., places + 1]
            code = (half * 2**14 // 2**16 % 2**16 + half * 2**14 % 2**16) // 16 ** (dim % 8 // 2) % 16 - 8
            out[..., dim] = (code * scales[:, :, dim // 16]).transpose(1, 2)
        found.append(out)
    return found


def _exact_rotated(rows: torch.Tensor, norm, rope: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    x = rows.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * norm.double()
    cos, sin = rope[0, positions].double()[:, None], rope[1, positions].double()[:, None]
    low, high = x[..., :32], x[..., 32:]
    return torch.cat((low * cos - high * sin, high * cos + low * sin), -1)


def _exact_new(state: dict, index: int, layer: int, positions: torch.Tensor):
    """The values of the new tokens' K and V [tokens, heads, 64] once they are in the cache."""
    norm = state["key_norm"][layer] if state["case"]["norm"] else None
    key = _exact_rotated(state["key"][index], norm, state["rope"], positions)
    return _exact_rounded(key), _exact_rounded(state["value"][index].double())


def _exact_write(state: dict):
    begin, found = LAYERS - state["case"]["layers"], []
    place = {int(b): i for i, b in enumerate(state["written"].tolist())}
    slots = state["slots"].tolist()
    row = torch.tensor([place[s // BLOCK] for s in slots], device=state["slots"].device)
    for layer in range(begin, LAYERS):
        key, value = _exact_stored(state, layer, state["written"].long())
        new_key, new_value = _exact_new(state, layer - begin, layer, state["positions"].long())
        key[row, state["slots"].long() % BLOCK] = new_key
        value[row, state["slots"].long() % BLOCK] = new_value
        found.append((key, value))
    return found


def _exact_one(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, start: int) -> torch.Tensor:
    """Causal attention of query [rows, 32, 64] at positions start, start + 1, ... of one request."""
    out = torch.empty_like(query)
    positions = start + torch.arange(query.shape[0], device=query.device)
    later = torch.arange(key.shape[0], device=query.device) > positions[:, None]
    for head in range(QUERY_HEADS):
        k, v = key[:, head // GROUP], value[:, head // GROUP]
        scores = (query[:, head] @ k.T / 8.0).masked_fill(later, -math.inf)
        out[:, head] = torch.softmax(scores, -1) @ v
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(state)
    norm = state["query_norm"][LAYER] if case.get("norm") else None
    flat = state["flat"].long()
    if case["op"] == "prompt":
        start, at, end = case["start"], state["positions"].long(), case["start"] + case["tokens"]
        stored = [x.flatten(0, 1) for x in _exact_stored(state, LAYER, flat)]  # [positions, heads, 64]
        for whole, new in zip(stored, _exact_new(state, 0, LAYER, at)):
            whole[start:end] = new
        query = _exact_rotated(state["query"], norm, state["rope"], at)
        out = _exact_one(query, stored[0][:end], stored[1][:end], start)
        return out, tuple(x.unflatten(0, (-1, BLOCK))[start // BLOCK :] for x in stored)
    prefix, lengths = state["prefix"].tolist(), state["lengths"].tolist()
    fresh, query = None, state["query"].double()
    if case["op"] == "decode":
        positions = state["lengths"].long() - 1
        fresh = _exact_new(state, 0, LAYER, positions)
        query = _exact_rotated(state["query"], norm, state["rope"], positions)
    outs, keys, values = [], [], []
    for b, length in enumerate(lengths):
        key, value = _exact_stored(state, LAYER, flat[prefix[b] : prefix[b + 1]])
        if fresh is not None:
            key[-1, (length - 1) % BLOCK], value[-1, (length - 1) % BLOCK] = fresh[0][b], fresh[1][b]
            keys.append(key[-1])
            values.append(value[-1])
        k, v = (x.flatten(0, 1)[:length].transpose(0, 1) for x in (key, value))
        scores = query[b].view(KV_HEADS, GROUP, HEAD_DIM) @ k.transpose(1, 2) / 8.0
        outs.append((torch.softmax(scores, -1) @ v).reshape(QUERY_HEADS, HEAD_DIM))
    if fresh is None:
        return torch.stack(outs)
    return torch.stack(outs), (torch.stack(keys), torch.stack(values))
