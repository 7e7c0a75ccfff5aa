"""What a configuration asks of its layers' windows, and what it may not leave unsaid."""

import json
import warnings

import pytest
import torch

from babyvllm.config import ModelConfig

HF = dict(architectures=["Qwen2ForCausalLM"], vocab_size=100, hidden_size=128, intermediate_size=256, num_hidden_layers=4,
          num_attention_heads=2, num_key_value_heads=1, rms_norm_eps=1e-6, max_position_embeddings=256, rope_theta=10000.0)


def test_first_tokens_without_a_window_are_refused():
    from babyvllm.layers.attention import Attention
    from babyvllm.models.qwen2 import Qwen2ForCausalLM

    with pytest.raises(ValueError, match="window"):
        Attention(2, 64, 1, sinks=4)
    cfg = ModelConfig(100, 128, 256, 1, 2, 1, 1e-6, 256, 10000.0, True, attention_sinks=4)
    with torch.device("meta"), pytest.raises(ValueError, match="window"):
        Qwen2ForCausalLM(cfg)
    assert Attention(2, 64, 1, window=8, sinks=4).sinks == 4 and Attention(2, 64, 1).window is None


def from_hf(tmp_path, **k):
    (tmp_path / "config.json").write_text(json.dumps({**HF, **k}))
    return ModelConfig.from_hf(str(tmp_path))


@pytest.mark.parametrize("given,window", [
    (dict(), None),
    (dict(sliding_window=64), None),  # named, not used
    (dict(use_sliding_window=False, sliding_window=64, max_window_layers=0), None),
    (dict(use_sliding_window=True, sliding_window=None, max_window_layers=0), None),
    (dict(use_sliding_window=True, sliding_window=64, max_window_layers=4), None),  # in no layer
    (dict(use_sliding_window=True, sliding_window=64, max_window_layers=9), None),
    (dict(use_sliding_window=True, sliding_window=64, max_window_layers=0), 64),
    (dict(use_sliding_window=True, sliding_window=64, layer_types=["sliding_attention"] * 4), 64),
    (dict(use_sliding_window=True, sliding_window=64, layer_types=["full_attention"] * 4), None),
    (dict(use_sliding_window=True, sliding_window=256, max_window_layers=0), None),  # hides no key
    (dict(use_sliding_window=True, sliding_window=255, max_window_layers=0), 255),
    (dict(use_sliding_window=True, sliding_window=64), None),  # 28 layers without by default
], ids=str)
def test_the_window_of_a_checkpoint(tmp_path, given, window):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cfg = from_hf(tmp_path, **given)
    assert cfg.sliding_window == window and cfg.attention_sinks == 0 and cfg.qk_norm is False


@pytest.mark.parametrize("given", [
    dict(max_window_layers=2), dict(layer_types=["full_attention", "sliding_attention"] * 2),
], ids=str)
def test_a_window_in_some_layers_is_not_dropped_without_a_word(tmp_path, given):
    with pytest.warns(UserWarning, match="64"):
        cfg = from_hf(tmp_path, use_sliding_window=True, sliding_window=64, **given)
    assert cfg.sliding_window is None
