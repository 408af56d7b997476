"""Operators of the transformer encoder that makes the token vectors: what a
late-interaction model runs in front of :func:`fused_head.maxsim_from_hidden`."""

from __future__ import annotations

from .attention import attention, attention_varlen
from .gated_ffn import gated_ffn
from .int8 import dequantize_int8_per_token, linear_int8, quantize_int8_per_token
from .layer_norm import layer_norm
from .rotary import rotary, rotary_frequencies

__all__ = ["attention", "attention_varlen", "dequantize_int8_per_token", "gated_ffn", "layer_norm", "linear_int8",
           "quantize_int8_per_token", "rotary", "rotary_frequencies"]
