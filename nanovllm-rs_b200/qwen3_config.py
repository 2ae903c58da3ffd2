"""Qwen3 architecture shapes the benchmark and tests run (config.rs:5-27).

Plain data, no torch and no native library: the CPU measurements (the
oracle-driven reference arm of bench.py) import these shapes without loading
libnvkv.so.  nvkv.decoder re-exports them.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional


@dataclass(frozen=True)
class RopeScaling:
    """How rotary frequencies are scaled for contexts past those of training
    (nvkv.rope_frequencies): kind "plain", "linear", "ntk", "yarn" or "bands".
    The reference has plain frequencies only (rotary_embedding.rs:28-57)."""

    kind: str
    factor: float = 1.0
    original_max_position: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    attention_factor: float = 0.0  # 0: the kind's own


@dataclass(frozen=True)
class Qwen3Config:
    """The config.json fields the reference reads (config.rs:5-27)."""

    hidden_size: int
    num_hidden_layers: int
    num_attention_heads: int
    num_key_value_heads: int
    intermediate_size: int
    vocab_size: int = 151936
    head_dim: int = 128
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1e6
    max_position_embeddings: int = 40960
    tie_word_embeddings: bool = False
    rope_scaling: Optional[RopeScaling] = None  # None: the reference's rotation


QWEN3_0_6B = Qwen3Config(1024, 28, 16, 8, 3072, tie_word_embeddings=True)
QWEN3_4B = Qwen3Config(2560, 36, 32, 8, 9728, tie_word_embeddings=True)
QWEN3_8B = Qwen3Config(4096, 36, 32, 8, 12288)
QWEN3_32B = Qwen3Config(5120, 64, 64, 8, 25600)
