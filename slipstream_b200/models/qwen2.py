"""Builder of the Qwen2.5 dense decoder from ``Qwen2Config``: which parts stand in
which layer, with which constants and tensor names.

Structure and names follow slipstream/models/causal_lm.py:31-141: per layer
``input_layernorm``, ``self_attn`` (biased q/k/v, unbiased o_proj:
slipstream/models/layers/attention.py:91-95), ``post_attention_layernorm``,
``mlp``; then ``model.norm`` and ``lm_head`` (the embedding matrix when tied).
``quantization`` "int8" or "fp8" builds the layers from the 8-bit parts; embedding, final norm and head stay as they are.
"""

from __future__ import annotations

from slipstream_b200.config.model_config import Qwen2Config
from slipstream_b200.parts import (Fp8PagedAttention, Fp8RMSNorm, Fp8SwiGLUFeedForward, Int8PagedAttention, Int8RMSNorm,
                                   Int8SwiGLUFeedForward, LMHead, PagedAttention, PreNormBlock, RMSNorm, RotaryEncoding,
                                   SwiGLUFeedForward, TokenEmbedding)

from .decoder import DecoderLM

_LAYERS = {None: (PagedAttention, SwiGLUFeedForward, RMSNorm),
           "int8": (Int8PagedAttention, Int8SwiGLUFeedForward, Int8RMSNorm),
           "fp8": (Fp8PagedAttention, Fp8SwiGLUFeedForward, Fp8RMSNorm)}


def build_qwen2(config: Qwen2Config, quantization: str | None = None) -> DecoderLM:
    c = config
    mixer, feed_forward, norm = _LAYERS[quantization]
    blocks = []
    rotary = RotaryEncoding(c.head_dim, c.rope_theta)  # one table of frequencies for all layers
    for i in range(c.num_hidden_layers):
        prefix = f"model.layers.{i}"
        attention = mixer(
            f"{prefix}.self_attn", c.hidden_size, c.num_attention_heads, c.num_key_value_heads, c.head_dim,
            rotary, qkv_bias=c.attention_bias, out_bias=False, window=None)
        ffn = feed_forward(f"{prefix}.mlp", c.hidden_size, c.intermediate_size, bias=c.mlp_bias)
        blocks.append(PreNormBlock(
            attention, ffn,
            norm(f"{prefix}.input_layernorm", c.hidden_size, c.rms_norm_eps),
            norm(f"{prefix}.post_attention_layernorm", c.hidden_size, c.rms_norm_eps)))
    return DecoderLM(
        c,
        TokenEmbedding("model.embed_tokens", c.vocab_size, c.hidden_size),
        blocks,
        RMSNorm("model.norm", c.hidden_size, c.rms_norm_eps),
        LMHead("lm_head", c.vocab_size, c.hidden_size,
               tied_to="model.embed_tokens.weight" if c.tie_word_embeddings else None))
