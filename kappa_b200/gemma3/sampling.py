"""Tokens from logits (kappa/gemma3/sampling.py): the same function as Qwen3's."""

from __future__ import annotations

from kappa_b200.qwen3.sampling import sample_tokens

__all__ = ["sample_tokens"]
