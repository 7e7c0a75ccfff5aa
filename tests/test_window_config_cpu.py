"""What a configuration asks of its layers' windows, and what it may not leave unsaid."""

import pytest
import torch

from babyvllm.config import ModelConfig

def test_first_tokens_without_a_window_are_refused():
    from babyvllm.layers.attention import Attention
    from babyvllm.models.qwen2 import Qwen2ForCausalLM

    with pytest.raises(ValueError, match="window"):
        Attention(2, 64, 1, sinks=4)
    cfg = ModelConfig(100, 128, 256, 1, 2, 1, 1e-6, 256, 10000.0, True, attention_sinks=4)
    with torch.device("meta"), pytest.raises(ValueError, match="window"):
        Qwen2ForCausalLM(cfg)
    assert Attention(2, 64, 1, window=8, sinks=4).sinks == 4 and Attention(2, 64, 1).window is None
