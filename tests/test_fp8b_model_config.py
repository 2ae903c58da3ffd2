"""The decoder's pool formats and scaled rotary frequencies, as far as they go
without a GPU: shapes, frequencies, refusals."""
from dataclasses import replace

import pytest
import torch

from nvkv import ops
from nvkv.decoder import QWEN3_0_6B, Qwen3TP, RopeScaling

SMALL = replace(QWEN3_0_6B, hidden_size=256, num_hidden_layers=1, num_attention_heads=4,
                num_key_value_heads=2, intermediate_size=128, vocab_size=64)


def _model(**kw):
    return Qwen3TP(replace(SMALL, **kw), seed=1, device="cpu", dtype=torch.bfloat16)


def test_block_scaled_pool_shapes():
    m = _model()
    m.allocate_kv_cache(3, 256, kv_fp8b=True)
    assert m.kv_fp8b and not m.kv_fp8
    assert m.k_caches[0].shape == (3, 256, 2, 128) and m.k_caches[0].dtype == torch.uint8
    assert m.kv_scales[0].shape == (3, 2, 16, 2) and m.kv_scales[0].dtype == torch.float32
    m.allocate_kv_cache(3, 256)
    assert not m.kv_fp8b and m.k_caches[0].dtype == torch.bfloat16


def test_frequencies_follow_the_config():
    want, _ = ops.rope_frequencies(128, 1e6, "plain")
    assert torch.equal(_model().inv_freq, want) and _model().rope_factor == 1.0
    m = _model(rope_scaling=RopeScaling("yarn", 4.0, 32768))
    want, a = ops.rope_frequencies(128, 1e6, "yarn", 4.0, 32768)
    assert torch.equal(m.inv_freq, want) and m.rope_factor == a > 1


def test_row_scaled_pool_refuses_what_it_cannot_do():
    with pytest.raises(ValueError):
        _model().allocate_kv_cache(2, 256, kv_fp8=True, kv_fp8b=True)
    with pytest.raises(ValueError):
        _model(rope_scaling=RopeScaling("linear", 2.0)).allocate_kv_cache(2, 256, kv_fp8=True)
