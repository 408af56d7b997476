"""Operators of the transformer encoder that makes the token vectors: what a
late-interaction model runs in front of :func:`fused_head.maxsim_from_hidden`."""

from __future__ import annotations

from .attention import attention, attention_varlen
from .gated_ffn import gated_ffn
from .layer_norm import layer_norm

__all__ = ["attention", "attention_varlen", "gated_ffn", "layer_norm"]
