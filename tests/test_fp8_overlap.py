"""Rotated queries written over themselves or over one another."""

from __future__ import annotations

import pytest
import torch

from pagedcore_b200 import fp8

ROW = 32 * 64


@pytest.mark.parametrize("strides, layers, tokens, apart", [
    ((6 * ROW, ROW), 2, 6, True), ((6 * ROW, ROW), 2, 7, False), ((ROW, 2 * ROW), 2, 6, True), ((ROW, 2 * ROW), 3, 6, False),
    ((ROW, ROW), 2, 2, False), ((ROW, ROW), 1, 9, True), ((0, ROW), 1, 9, True), ((0, ROW), 2, 9, False), ((ROW, 8), 4, 1, True),
    ((ROW, 8), 4, 2, False), ((3 * ROW + 128, ROW + 64), 2, 3, True), ((3 * ROW + 64, ROW + 64), 2, 3, False), ((8, 8), 1, 1, True),
])
def test_rows_apart(strides, layers, tokens, apart) -> None:
    assert fp8._rows_apart((*strides, 64, 1), layers, tokens) is apart
    covered = torch.zeros((layers + tokens) * 9 * ROW, dtype=torch.int8)  # the same by writing every row
    for layer in range(layers):
        for token in range(tokens):
            at = layer * strides[0] + token * strides[1]
            covered[at : at + ROW] += 1
    assert (int(covered.max()) == 1) is apart


def test_queries_that_an_output_overlaps_are_found() -> None:
    base = torch.zeros(12 * ROW, dtype=torch.float16)
    rows = lambda first, count, stride=ROW: base.as_strided((1, count, 32, 64), (count * stride, stride, 64, 1), first)  # noqa: E731
    assert not fp8._mixes(rows(0, 4), rows(0, 4))
    assert not fp8._mixes(rows(0, 4), rows(4 * ROW, 4)) and not fp8._mixes(rows(4 * ROW, 4), rows(0, 4))
    assert fp8._mixes(rows(0, 4), rows(ROW, 4)) and fp8._mixes(rows(ROW, 4), rows(64, 4))
    assert fp8._mixes(rows(0, 4), rows(0, 4, 2 * ROW))
    assert fp8._mixes(rows(0, 4), base[: 8 * ROW].view(torch.float32).view(1, 4, 32, 64))


@pytest.mark.gpu
def test_a_query_rotated_over_its_neighbours_is_rotated_right() -> None:
    from tests.test_fp8_gpu import LAYER, CacheCase, randn

    case = CacheCase(181, [0], spare=30)
    case.tables[0] += [case.free.pop() for _ in range(25)]
    tokens = 400
    key, value, query = (randn(182 + heads, 1, tokens, heads, 64).half() for heads in (4, 5, 32))
    value = value[:, :, :4]
    arguments = dict(layer_begin=LAYER, error_flag=case.flag, rope_table=case.rope,
                     positions=torch.arange(tokens, dtype=torch.int32, device=case.device))
    slots = torch.tensor(case.slots(0, 0, tokens), dtype=torch.int32, device=case.device)
    expected = torch.empty_like(query)
    fp8.append_kv(case.cache, key, value, slots, query=query, query_out=expected, **arguments)
    for shift in (0, ROW, -ROW, 64, 3 * ROW + 8):
        base = torch.zeros((tokens + 12) * ROW, dtype=torch.float16, device=case.device)
        view = lambda at: base[at : at + tokens * ROW].view(1, tokens, 32, 64)  # noqa: E731
        source = view(5 * ROW).copy_(query)
        assert torch.equal(fp8.append_kv(case.cache, key, value, slots, query=source, query_out=view(5 * ROW + shift), **arguments), expected)
    both = torch.zeros(2, tokens, 32, 64, dtype=torch.float16, device=case.device)
    two = lambda t: t.expand(2, *t.shape[1:])  # noqa: E731
    with pytest.raises(ValueError, match="query_out"):
        fp8.append_kv(case.cache, two(key), two(value), slots, query=two(query), query_out=both.as_strided((2, tokens, 32, 64), (ROW, ROW, 64, 1)),
                      **(arguments | {"layer_begin": 0}))
    for out in (both, torch.zeros(tokens, 2, 32, 64, dtype=torch.float16, device=case.device).transpose(0, 1)):
        fp8.append_kv(case.cache, two(key), two(value), slots, query=two(query), query_out=out, **(arguments | {"layer_begin": 0}))
        assert torch.equal(out[0], expected[0]) and torch.equal(out[1], expected[0])
    assert int(case.flag.item()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows, dim", [(3, 200), (64, 2048), (5, 4104), (9, 8192)])
def test_a_norms_residual_may_be_either_input(rows, dim) -> None:
    from tests.test_fp8_gpu import randn

    weight = randn(190, dim).half()
    hidden, delta = randn(191, rows, dim).half(), randn(192, rows, dim).half()
    expected = torch.empty_like(hidden)
    out = fp8.add_rms_norm(hidden, delta, weight, residual=expected)
    for which in (0, 1):
        inputs = [hidden.clone(), delta.clone()]
        again = fp8.add_rms_norm(*inputs, weight, residual=inputs[which])
        assert torch.equal(inputs[which], expected) and torch.equal(inputs[1 - which], (hidden, delta)[1 - which])
        assert torch.equal(again.codes.view(torch.uint8), out.codes.view(torch.uint8)) and torch.equal(again.scales, out.scales)


@pytest.mark.gpu
def test_a_chain_of_early_launches_reads_what_was_just_written() -> None:
    """Norm, product, SwiGLU and product again in the same storage, step after step, back to back and apart."""
    from tests.test_fp8_gpu import randn

    weight = torch.ones(512, dtype=torch.float16, device="cuda")
    up, down = fp8.quantize_weight(0.05 * randn(193, 2048, 512)), fp8.quantize_weight(0.05 * randn(194, 512, 1024))

    def chain(hidden: torch.Tensor, steps: int, wait: bool) -> torch.Tensor:
        hidden = hidden.clone()
        delta = torch.zeros_like(hidden)
        for _ in range(steps):
            rows = fp8.add_rms_norm(hidden, delta, weight)
            if wait:
                torch.cuda.synchronize()
            gate_up = fp8.linear(rows, up)
            if wait:
                torch.cuda.synchronize()
            act = fp8.silu_mul(gate_up)
            if wait:
                torch.cuda.synchronize()
            fp8.linear(act, down, delta)
            if wait:
                torch.cuda.synchronize()
        return hidden

    for count in (1, 20, 100, 700):
        hidden = randn(195 + count, count, 512).half()
        assert torch.equal(chain(hidden, 30, False), chain(hidden, 30, True))
