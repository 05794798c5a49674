"""The batched decoder with 8-bit projections.

``Fp8BatchedDecoder`` is :class:`pagedcore_b200.decoder.BatchedDecoder` with the
Q/K/V, output, gate/up and down projections of every layer in E4M3: weights
with a scale per 128 x 128 block, made once here, and activations with a scale
per row and 128 values, made by the kernel before each projection (the
residual add + RMSNorm, SwiGLU's product, or a conversion of the attention).
The residual stream, the embedding, the final norm and the LM head stay FP16.
It runs over either allocator, an ``Fp8KVAllocator`` included, and through the
step graphs.
"""

from __future__ import annotations

from collections.abc import Callable

import torch
import torch.nn.functional as F
from torch import Tensor

from pagedcore_b200 import fp8, kernels
from pagedcore_b200.decoder import BatchedDecoder
from pagedcore_b200.weights import HEAD_DIM, HIDDEN, KV_HEADS, LAYERS, QUERY_HEADS, TinyLlamaWeights


class Fp8BatchedDecoder(BatchedDecoder):
    """Batched decode steps and prompt prefill over 8-bit copies of a set of weights."""

    def __init__(self, weights: TinyLlamaWeights) -> None:
        if len(weights.layers) != LAYERS:
            raise ValueError("paged decode requires 22 decoder layers")
        self.weights = weights
        quantize = fp8.quantize_weight
        self.qkv = [quantize(torch.cat((layer.q_proj, layer.k_proj, layer.v_proj))) for layer in weights.layers]
        self.output = [quantize(layer.o_proj) for layer in weights.layers]
        self.gate_up = [quantize(torch.cat((layer.gate_proj, layer.up_proj))) for layer in weights.layers]
        self.down = [quantize(layer.down_proj) for layer in weights.layers]
        if weights.embedding.is_cuda:
            kernels.linear_error_flag(weights.embedding.device)  # before any graph capture

    def forward(self, input_ids: Tensor, attend: Callable[[int, Tensor, Tensor, Tensor], Tensor]) -> Tensor:
        """The decoder stack for token ids [B, 1], as ``BatchedDecoder.forward``."""
        weights = self.weights
        batch = input_ids.shape[0]
        q_width, kv_width = QUERY_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
        hidden = F.embedding(input_ids, weights.embedding).view(batch, HIDDEN)  # updated in place
        delta = None  # the output still to be added to the residual stream
        for index, layer in enumerate(weights.layers):
            qkv = fp8.linear(fp8.add_rms_norm(hidden, delta, layer.input_norm), self.qkv[index])
            query = qkv[:, :q_width].view(batch, QUERY_HEADS, HEAD_DIM)
            key = qkv[:, q_width : q_width + kv_width].view(batch, KV_HEADS, HEAD_DIM)
            value = qkv[:, q_width + kv_width :].view(batch, KV_HEADS, HEAD_DIM)
            attention = attend(index, query, key, value)
            delta = fp8.linear(fp8.quantize_rows(attention.reshape(batch, HIDDEN)), self.output[index])
            gate_up = fp8.linear(fp8.add_rms_norm(hidden, delta, layer.post_attention_norm), self.gate_up[index])
            delta = fp8.linear(fp8.silu_mul(gate_up), self.down[index])
        x = torch.empty_like(hidden)
        kernels.add_rms_norm(hidden, delta, weights.final_norm, x)
        return kernels.linear(x, weights.lm_head).view(batch, 1, -1)
