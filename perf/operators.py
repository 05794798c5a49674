"""What the 8-bit operators cost: cases, inputs, plain forms and 64-bit results.

Four operators of the 8-bit decode path, each as a user's program calls it:

- ``norm``    residual add + RMSNorm with its output in 8 bits, a scale per row
  and block of 128 values; the 8-bit rows come back as the values they stand for.
- ``linear``  a projection of 8-bit rows by 8-bit weights (a scale per 128 x 128
  block), FP16 out.
- ``decode``  one decode layer over an 8-bit KV cache with a scale per block of 16
  tokens and head: the new token's K (rotated) and V written, then attention.
- ``prompt``  one layer of a prompt chunk over the same cache: K/V written, then
  causal attention through the block table.

8 bits are E4M3.  A scale made here is the smallest power of two, between 2^-15 and
2^8, that brings the block's largest magnitude to 448 or less.
"""

from __future__ import annotations

import math

import torch

own = False

LAYERS, LAYER = 2, 1  # the cache holds two layers; the second is used
KV_HEADS, GROUP, HEAD_DIM, BLOCK = 4, 8, 64, 16
QUERY_HEADS = KV_HEADS * GROUP
CONTEXT = 2048
EPS = 1e-5


def listed() -> list[dict]:
    return [
        # The smallest calls: one sequence decoding, bound by launch latency.
        {"name": "norm_row", "op": "norm", "rows": 1, "dim": 2048, "delta": True},
        # A decode batch of this repository's benchmark (256 sequences).
        {"name": "norm_batch", "op": "norm", "rows": 256, "dim": 2048, "delta": True},
        # The rows of a full-length prompt.
        {"name": "norm_prompt", "op": "norm", "rows": 2047, "dim": 2048, "delta": True},
        # Q/K/V projection of one sequence.
        {"name": "linear_row", "op": "linear", "rows": 1, "n": 2560, "k": 2048},
        # Down projection of a small decode batch: few output tiles, long sums.
        {"name": "linear_small_batch", "op": "linear", "rows": 32, "n": 2048, "k": 5632},
        # Gate and up projections of the benchmark's decode batch.
        {"name": "linear_batch", "op": "linear", "rows": 256, "n": 11264, "k": 2048},
        # The same projections for a prompt: bound by the tensor cores.
        {"name": "linear_prompt", "op": "linear", "rows": 2047, "n": 11264, "k": 2048},
        # One short sequence: a single partial block and its first neighbour.
        {"name": "decode_one", "op": "decode", "batch": 1, "low": 17, "high": 17},
        # A few sequences at the context limit: the long axis has to be split.
        {"name": "decode_few_long", "op": "decode", "batch": 3, "low": 2048, "high": 2048},
        # The benchmark's ragged batch: 256 sequences of 1 to 2048 tokens.
        {"name": "decode_batch", "op": "decode", "batch": 256, "low": 1, "high": 2048},
        # A short prompt continuing a cached conversation inside a block.
        {"name": "prompt_continued", "op": "prompt", "start": 601, "tokens": 75},
        # A full-length prompt.
        {"name": "prompt_full", "op": "prompt", "start": 0, "tokens": 2047},
    ]


def _log(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "linear", "decode", "prompt"))
    if op == "norm":
        dim = 8 * _log(rng, 8, 1024)
        rows = _log(rng, 1, max(1, min(4096, 2047 * 2048 // dim)))
        return {"op": op, "rows": rows, "dim": dim, "delta": rng.random() < 0.8}
    if op == "linear":
        n, k = _log(rng, 33, 11264), 16 * _log(rng, 1, 352)
        return {"op": op, "rows": _log(rng, 1, min(2047, 2047 * 11264 * 2048 // (n * k))), "n": n, "k": k}
    if op == "decode":
        high = _log(rng, 1, CONTEXT)
        return {"op": op, "batch": _log(rng, 1, 256), "low": rng.randint(1, high), "high": high}
    tokens = _log(rng, 1, 1500)
    return {"op": op, "start": rng.randint(0, 2047 - tokens), "tokens": tokens}


# -- inputs ----------------------------------------------------------------------
def _exponent(amax: torch.Tensor) -> torch.Tensor:
    """log2 of the scale of a block whose largest magnitude is ``amax`` (float32)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    needed = exponent - 9 + (mantissa > 0.875).int()  # 448 = 0.875 * 2^9
    return torch.where(amax > 0, needed, -15).clamp(-15, 8)


def _encode(scaled: torch.Tensor) -> torch.Tensor:
    return scaled.to(torch.float8_e4m3fn)


def _power(exponent: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones_like(exponent, dtype=torch.float32), exponent)


def _groups(values: torch.Tensor) -> torch.Tensor:
    """[rows, width] -> [rows, blocks, 128], the last block filled with zeros."""
    rows, width = values.shape
    blocks = -(-width // 128)
    return torch.nn.functional.pad(values, (0, 128 * blocks - width)).view(rows, blocks, 128)


def _quantize_rows(values: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 [rows, width] -> E4M3 codes [rows, width] and scales [rows, ceil(width / 128)]."""
    grouped = _groups(values)
    scale = _power(_exponent(grouped.abs().amax(-1)))
    codes = _encode(grouped / scale[..., None]).view(torch.uint8)
    return codes.flatten(1)[:, : values.shape[1]].contiguous().view(torch.float8_e4m3fn), scale


def _rope_table(device) -> torch.Tensor:
    """FP16 cos and sin [2, 2048, 32]."""
    inverse = 1.0 / (10000.0 ** (torch.arange(0, HEAD_DIM, 2).float() / HEAD_DIM))
    angles = torch.arange(CONTEXT).float()[:, None] * inverse
    return torch.stack((angles.cos(), angles.sin())).half().to(device)


def _history(generator, blocks: int, device) -> dict:
    """A filled cache [layers, blocks, heads, ...]: K tiles [16, 64], V tiles [64, 16] and their scales."""

    def tiles(shape, spread):
        values = torch.randn((LAYERS, blocks, KV_HEADS, *shape), device=device, generator=generator) * spread
        scale = _power(_exponent(values.abs().amax((-2, -1))))
        return _encode(values / scale[..., None, None]), scale

    channels = 0.5 + 2.5 * torch.rand((HEAD_DIM,), device=device, generator=generator) ** 4  # a few strong K channels
    key_codes, key_scales = tiles((BLOCK, HEAD_DIM), channels)
    value_codes, value_scales = tiles((HEAD_DIM, BLOCK), 1.0)
    return {"key_codes": key_codes, "key_scales": key_scales, "value_codes": value_codes, "value_scales": value_scales}


def _clear(state: dict, block: torch.Tensor, used: torch.Tensor) -> None:
    """Zero codes in the never-written slots (``used`` and later) of ``block``; scale 1 where none was written."""
    slot = torch.arange(BLOCK, device=block.device)
    keep = slot < used[:, None]  # [blocks, 16]
    for name, mask in (("key", keep[:, None, :, None]), ("value", keep[:, None, None, :])):
        codes = state[name + "_codes"].view(torch.uint8)
        codes[:, block] = codes[:, block] * mask
        scales = state[name + "_scales"]
        scales[:, block] = torch.where(used[:, None] > 0, scales[:, block], 1.0)


def _lengths(case: dict) -> list[int]:
    batch, low, high = case["batch"], case["low"], case["high"]
    return [low + (high - low) * i // max(1, batch - 1) for i in range(batch)]


def prepare(case: dict, seed: int) -> dict:
    device = torch.device("cuda")
    generator = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=device, generator=generator)

    state = {"case": case}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        state["hidden"] = (3 * normal(rows, dim)).half()
        state["delta"] = normal(rows, dim).half() if case["delta"] else None
        state["weight"] = (1 + 0.1 * normal(dim)).half()
        state["residual"] = torch.empty_like(state["hidden"])
        return state
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        state["x_codes"], state["x_scales"] = _quantize_rows(normal(rows, k) * torch.exp(normal(rows, 1)))
        weight = 0.02 * normal(n, k)
        tall, wide = -(-n // 128), -(-k // 128)
        padded = torch.zeros(128 * tall, 128 * wide, device=device)
        padded[:n, :k] = weight
        blocks = padded.view(tall, 128, wide, 128)
        scales = blocks.abs().amax((1, 3)) / 448
        codes = _encode((blocks / scales[:, None, :, None]).clamp(-448, 448)).view(torch.uint8)
        codes = codes.reshape(128 * tall, 128 * wide)[:n, :k].contiguous()
        state["w_codes"], state["w_scales"] = codes.view(torch.float8_e4m3fn), scales.contiguous()
        return state

    lengths = _lengths(case) if case["op"] == "decode" else [case["start"] + case["tokens"]]
    counts = [-(-length // BLOCK) for length in lengths]
    total = sum(counts)
    state |= _history(generator, total + 3, device)
    state["flat"] = torch.randperm(total + 3, device=device, generator=generator)[:total].int()
    state["total_blocks"] = total
    state["rope"] = _rope_table(device)
    state["error_flag"] = torch.zeros(1, dtype=torch.int32, device=device)
    if case["op"] == "decode":
        order = torch.randperm(len(lengths), device=device, generator=generator)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)[order]
        blocks = torch.tensor(counts, dtype=torch.int32, device=device)[order]
        state["prefix"] = torch.nn.functional.pad(torch.cumsum(blocks, 0), (1, 0)).int()
        state["last"] = state["flat"][(state["prefix"][1:] - 1).long()]
        _clear(state, state["last"].long(), (state["lengths"].long() - 1) % BLOCK)
        rows = len(lengths)
    else:
        start, rows = case["start"], case["tokens"]
        state["positions"] = torch.arange(start, start + rows, dtype=torch.int32, device=device)
        positions = state["positions"].long()
        state["slots"] = state["flat"][positions // BLOCK] * BLOCK + state["positions"] % BLOCK
        state["written"] = state["flat"][start // BLOCK :].contiguous()
        used = (start - BLOCK * torch.arange(start // BLOCK, total, device=device)).clamp(0, BLOCK)
        _clear(state, state["written"].long(), used)
    state["query"] = normal(rows, QUERY_HEADS, HEAD_DIM).half()
    state["key"] = (normal(rows, KV_HEADS, HEAD_DIM) * 1.2).half()
    state["value"] = normal(rows, KV_HEADS, HEAD_DIM).half()
    return state


# -- plain forms ---------------------------------------------------------------------
def _norm(state: dict):
    hidden = state["hidden"].float()
    if state["delta"] is not None:
        hidden = hidden + state["delta"].float()
    scaled = hidden * torch.rsqrt((hidden * hidden).mean(-1, keepdim=True) + EPS) * state["weight"].float()
    codes, scales = _quantize_rows(scaled)
    values = _groups(codes.float()) * scales[..., None]
    return values.flatten(1)[:, : scaled.shape[1]].half(), hidden.half()


def _linear(state: dict):
    k = state["x_codes"].shape[1]
    x = (_groups(state["x_codes"].float()) * state["x_scales"][..., None]).flatten(1)[:, :k]
    n = state["w_codes"].shape[0]
    scales = state["w_scales"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return (x @ (state["w_codes"].float() * scales).T).half()


def _rotate(tensor: torch.Tensor, state: dict, positions: torch.Tensor) -> torch.Tensor:
    """RoPE of [rows, heads, 64] at int64 positions [rows], in float32."""
    cos, sin = (table[positions].float().repeat(1, 2)[:, None] for table in state["rope"])
    x = tensor.float()
    turned = torch.cat((-x[..., 32:], x[..., :32]), -1)
    return x * cos + turned * sin


def _write(state: dict, name: str, blocks: torch.Tensor, tiles: torch.Tensor, first: torch.Tensor, end: torch.Tensor):
    """Write slots [first, end) of each block from float32 ``tiles`` [blocks, heads, 16, 64].

    A block's first tokens set its scale; later ones raise it when they need more, and
    the codes already there are then rounded again to the larger scale.
    """
    slot = torch.arange(BLOCK, device=blocks.device)
    new = ((slot >= first[:, None]) & (slot < end[:, None]))[:, None, :, None]
    old = (slot < first[:, None])[:, None, :, None]
    codes, scales = state[name + "_codes"][LAYER], state[name + "_scales"][LAYER]
    stored = codes.view(torch.uint8)[blocks].view(torch.float8_e4m3fn)
    if name == "value":  # held as [64, 16]
        stored = stored.transpose(-1, -2)
    needed = _exponent(torch.where(new, tiles.abs(), 0.0).amax((-2, -1)))
    held = torch.frexp(scales[blocks])[1] - 1
    exponent = torch.where(first[:, None] > 0, torch.maximum(held, needed), needed)
    scale = _power(exponent)[..., None, None]
    again = stored.float() * (scales[blocks][..., None, None] / scale)
    largest = torch.where(exponent == 8, 240.0, 448.0)[..., None, None]
    fresh = torch.minimum(torch.maximum(tiles / scale, -largest), largest)
    written = torch.where(new, fresh, again)
    result = torch.where(new | old, _encode(written).view(torch.uint8), stored.contiguous().view(torch.uint8))
    if name == "value":
        result = result.transpose(-1, -2)
    codes.view(torch.uint8)[blocks] = result
    scales[blocks] = scale[..., 0, 0]


def _values(state: dict, name: str, blocks: torch.Tensor) -> torch.Tensor:
    """float32 [blocks..., heads, 16, 64] of the cache."""
    codes = state[name + "_codes"][LAYER].view(torch.uint8)[blocks].view(torch.float8_e4m3fn).float()
    values = codes * state[name + "_scales"][LAYER][blocks][..., None, None]
    return values.transpose(-1, -2) if name == "value" else values


def _softmax(scores: torch.Tensor) -> torch.Tensor:
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return weights / weights.sum(-1, keepdim=True)


def _read(state: dict, blocks: torch.Tensor):
    """K and V [blocks, 16, heads, 64] FP16 of the given blocks."""
    return tuple(_values(state, name, blocks).transpose(1, 2).half() for name in ("key", "value"))


def _decode(state: dict):
    lengths, prefix = state["lengths"].long(), state["prefix"].long()
    positions, last = lengths - 1, state["last"].long()
    slot = positions % BLOCK
    query = _rotate(state["query"], state, positions)
    key = _rotate(state["key"], state, positions)
    for name, token in (("key", key), ("value", state["value"].float())):
        _write(state, name, last, token[:, :, None].expand(-1, -1, BLOCK, -1), slot, slot + 1)
    batch = lengths.shape[0]
    most = int(-(-state["case"]["high"] // BLOCK))
    at = (prefix[:-1, None] + torch.arange(most, device=prefix.device)).clamp(max=state["total_blocks"] - 1)
    table = state["flat"].long()[at]  # [batch, most]
    keys = _values(state, "key", table).permute(0, 2, 1, 3, 4).reshape(batch, KV_HEADS, most * BLOCK, HEAD_DIM)
    scores = query.view(batch, KV_HEADS, GROUP, HEAD_DIM) @ keys.transpose(-1, -2) * HEAD_DIM**-0.5
    beyond = (torch.arange(most * BLOCK, device=lengths.device) >= lengths[:, None])[:, None, None]
    weights = _softmax(scores.masked_fill(beyond, -math.inf))
    values = _values(state, "value", table).permute(0, 2, 1, 3, 4).reshape(batch, KV_HEADS, most * BLOCK, HEAD_DIM)
    values = values.masked_fill(beyond.transpose(-1, -2), 0.0)
    out = (weights @ values).view(batch, QUERY_HEADS, HEAD_DIM).half()
    return out, _read(state, last)


def _prompt(state: dict):
    start, tokens = state["case"]["start"], state["case"]["tokens"]
    positions, written = state["positions"].long(), state["written"].long()
    query = _rotate(state["query"], state, positions)
    key = _rotate(state["key"], state, positions)
    count = written.shape[0]
    base = start // BLOCK * BLOCK
    first = (start - base - BLOCK * torch.arange(count, device=written.device)).clamp(0, BLOCK)
    end = (start + tokens - base - BLOCK * torch.arange(count, device=written.device)).clamp(0, BLOCK)
    for name, rows in (("key", key), ("value", state["value"].float())):
        tiles = torch.zeros((count * BLOCK, KV_HEADS, HEAD_DIM), device=rows.device)
        tiles[start - base : start - base + tokens] = rows
        _write(state, name, written, tiles.view(count, BLOCK, KV_HEADS, HEAD_DIM).transpose(1, 2), first, end)
    table = state["flat"].long()
    total = start + tokens
    keys, values = (
        _values(state, name, table).transpose(0, 1).reshape(KV_HEADS, -1, HEAD_DIM)[:, :total]
        for name in ("key", "value")
    )
    grouped = query.view(tokens, KV_HEADS, GROUP, HEAD_DIM).permute(1, 2, 0, 3)
    scores = grouped @ keys[:, None].transpose(-1, -2) * HEAD_DIM**-0.5
    beyond = torch.arange(total, device=table.device) > positions[:, None]
    out = _softmax(scores.masked_fill(beyond, -math.inf)) @ values[:, None]
    return out.permute(2, 0, 1, 3).reshape(tokens, QUERY_HEADS, HEAD_DIM).half(), _read(state, written)


def _run_own(state: dict):
    from pagedcore_b200 import fp8

    op = state["case"]["op"]
    if op == "norm":
        rows = fp8.add_rms_norm(state["hidden"], state["delta"], state["weight"], residual=state["residual"], eps=EPS)
        return rows.to_half(), state["residual"] if state["delta"] is not None else state["hidden"]
    if op == "linear":
        return fp8.linear(
            fp8.Fp8Rows(state["x_codes"], state["x_scales"]), fp8.Fp8Weight(state["w_codes"], state["w_scales"])
        )
    cache = fp8.Fp8Cache(state["key_codes"], state["value_codes"], state["key_scales"], state["value_scales"])
    if op == "decode":
        out = fp8.decode_layer(
            cache, LAYER, state["query"], state["key"], state["value"], state["rope"], state["lengths"],
            state["prefix"], state["flat"], state["total_blocks"], state["error_flag"],
        )
        return out, fp8.read_blocks(cache, LAYER, state["last"], state["error_flag"])
    query = fp8.append_kv(
        cache, state["key"][None], state["value"][None], state["slots"], layer_begin=LAYER,
        error_flag=state["error_flag"], positions=state["positions"], rope_table=state["rope"],
        query=state["query"][None],
    )
    out = fp8.prefill_attention(cache, LAYER, query[0], state["flat"], state["case"]["start"], state["error_flag"])
    return out, fp8.read_blocks(cache, LAYER, state["written"], state["error_flag"])


_PLAIN = {"norm": _norm, "linear": _linear, "decode": _decode, "prompt": _prompt}


def run(state: dict):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# -- what a pass cannot do without --------------------------------------------------------
def work(case: dict) -> dict:
    op = case["op"]
    if op == "norm":
        values = case["rows"] * case["dim"]
        # hidden in, the 8-bit values' FP16 form out; with delta: delta in and the sum out.
        return {"bytes": (8 if case["delta"] else 4) * values + 2 * case["dim"], "flops": 6 * values}
    if op == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        scales = 4 * (rows * -(-k // 128) + -(-n // 128) * -(-k // 128))
        return {"bytes": rows * k + n * k + 2 * rows * n + scales, "flops": 2 * rows * n * k}
    token = 2 * KV_HEADS * HEAD_DIM  # bytes of one token's K and V codes
    block = 2 * KV_HEADS * 4  # bytes of one block's scales
    if op == "decode":
        lengths = _lengths(case)
        tokens, blocks, rows = sum(lengths), sum(-(-n // BLOCK) for n in lengths), len(lengths)
        pairs, back = tokens, rows
        fresh = rows
    else:
        start, rows = case["start"], case["tokens"]
        tokens = start + rows
        blocks = -(-tokens // BLOCK)
        pairs = rows * start + rows * (rows + 1) // 2
        back = blocks - start // BLOCK
        fresh = rows
    heads = rows * HEAD_DIM * 2 * (2 * QUERY_HEADS + 2 * KV_HEADS)  # queries, outputs, new K and V
    return {
        "bytes": tokens * token + blocks * block + heads + fresh * token + back * BLOCK * token * 2,
        "flops": 4 * pairs * QUERY_HEADS * HEAD_DIM,
    }


# -- the same in 64 bits -------------------------------------------------------------------
def _exact_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two in [2^-15, 2^8] with amax / scale <= 448."""
    powers = 2.0 ** torch.arange(-15, 9, dtype=torch.float64, device=amax.device)
    fits = amax[..., None] <= 448 * powers
    first = torch.where(fits.any(-1), fits.double().argmax(-1), 23)
    return powers[first]


def _exact_round(values: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The nearest E4M3 multiple of ``scale`` (ties to even), in float64."""
    v = values / scale
    size = torch.floor(torch.log2(v.abs().clamp(min=2.0**-6)))
    step = 2.0 ** (size - 3)
    limit = torch.where(scale == 256.0, 240.0, 448.0).double()
    return torch.minimum(torch.maximum(torch.round(v / step) * step, -limit), limit) * scale


def _exact_norm(state: dict):
    x = state["hidden"].double()
    if state["delta"] is not None:
        x = x + state["delta"].double()
    y = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * state["weight"].double()
    out = torch.empty_like(y)
    for at in range(0, y.shape[1], 128):
        part = y[:, at : at + 128]
        out[:, at : at + 128] = _exact_round(part, _exact_scale(part.abs().amax(1, keepdim=True)))
    return out, x


def _exact_linear(state: dict):
    x, w = state["x_codes"].double(), state["w_codes"].double()
    out = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    for j, at in enumerate(range(0, x.shape[1], 128)):
        scaled = w[:, at : at + 128] * state["w_scales"][:, j].double().repeat_interleave(128)[: w.shape[0], None]
        out += state["x_scales"][:, j : j + 1].double() * (x[:, at : at + 128] @ scaled.T)
    return out


def _exact_rotate(rows: torch.Tensor, rope: torch.Tensor, positions) -> torch.Tensor:
    cos, sin = rope[0, positions].double()[:, None], rope[1, positions].double()[:, None]
    low, high = rows[..., :32].double(), rows[..., 32:].double()
    return torch.cat((low * cos - high * sin, high * cos + low * sin), -1)


def _exact_context(state: dict, table: torch.Tensor, name: str, start: int, rows: torch.Tensor) -> torch.Tensor:
    """One request's K or V [tokens, heads, 64] with ``rows`` [new, heads, 64] at ``start`` and later."""
    codes = state[name + "_codes"][LAYER].view(torch.uint8)[table].view(torch.float8_e4m3fn).double()
    if name == "value":
        codes = codes.transpose(-1, -2)
    scales = state[name + "_scales"][LAYER][table].double()  # [blocks, heads]
    old = (codes * scales[..., None, None]).transpose(1, 2).flatten(0, 1)[:start]  # [start, heads, 64]
    whole = torch.cat((old, rows))
    fresh = start // BLOCK  # the first block that is written
    count = whole.shape[0] - fresh * BLOCK
    tail = torch.zeros(-(-count // BLOCK) * BLOCK, KV_HEADS, HEAD_DIM, dtype=torch.float64, device=rows.device)
    tail[: start % BLOCK] = old[fresh * BLOCK :]
    new = tail.clone()
    new[start % BLOCK : count] = rows
    needed = new.clone()
    needed[: start % BLOCK] = 0
    scale = _exact_scale(needed.view(-1, BLOCK, KV_HEADS, HEAD_DIM).abs().amax((1, 3)))
    if start % BLOCK:
        scale[0] = torch.maximum(scale[0], scales[fresh])
    rounded = _exact_round(new.view(-1, BLOCK, KV_HEADS, HEAD_DIM), scale[:, None, :, None])
    return torch.cat((old[: fresh * BLOCK], rounded.flatten(0, 1)))  # whole blocks; the tail's free slots are zeros


def _exact_attend(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, start: int) -> torch.Tensor:
    """Causal attention of query [rows, 32, 64] at positions start, start + 1, ... of one request."""
    out = torch.empty_like(query)
    tokens = start + query.shape[0]
    for head in range(QUERY_HEADS):
        k, v = key[:tokens, head // GROUP], value[:tokens, head // GROUP]
        scores = query[:, head] @ k.T / 8.0
        later = torch.arange(tokens, device=query.device) > start + torch.arange(query.shape[0], device=query.device)[:, None]
        out[:, head] = torch.softmax(scores.masked_fill(later, -math.inf), -1) @ v
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(state)
    if case["op"] == "linear":
        return _exact_linear(state)
    flat = state["flat"].long()
    if case["op"] == "prompt":
        start, at = case["start"], state["positions"].long()
        key = _exact_context(state, flat, "key", start, _exact_rotate(state["key"], state["rope"], at))
        value = _exact_context(state, flat, "value", start, state["value"].double())
        out = _exact_attend(_exact_rotate(state["query"], state["rope"], at), key, value, start)
        written = tuple(x[start // BLOCK * BLOCK :].view(-1, BLOCK, KV_HEADS, HEAD_DIM) for x in (key, value))
        return out, written
    prefix, lengths = state["prefix"].tolist(), state["lengths"].tolist()
    outs, keys, values = [], [], []
    for b, length in enumerate(lengths):
        table, at = flat[prefix[b] : prefix[b + 1]], torch.tensor([length - 1], device=flat.device)
        key = _exact_context(state, table, "key", length - 1, _exact_rotate(state["key"][b : b + 1], state["rope"], at))
        value = _exact_context(state, table, "value", length - 1, state["value"][b : b + 1].double())
        query = _exact_rotate(state["query"][b : b + 1], state["rope"], at)[0].view(KV_HEADS, GROUP, HEAD_DIM)
        k, v = key[:length].transpose(0, 1), value[:length].transpose(0, 1)
        outs.append((torch.softmax(query @ k.transpose(1, 2) / 8.0, -1) @ v).reshape(QUERY_HEADS, HEAD_DIM))
        keys.append(key[-BLOCK:])
        values.append(value[-BLOCK:])
    return torch.stack(outs), (torch.stack(keys), torch.stack(values))
