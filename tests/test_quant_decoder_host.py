"""What a decoder layer refuses when it is made."""
import pytest
import torch

from quant_decoder import QuantDecoderLayer


def test_layers_that_attention_does_not_take():
    sizes = dict(heads=2, kv_heads=1, head_dim=64, hidden=32, device="cpu")
    QuantDecoderLayer(32, **sizes)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        QuantDecoderLayer(32, dtype=torch.float32, **sizes)
    with pytest.raises(ValueError, match="head dimension"):
        QuantDecoderLayer(32, **{**sizes, "head_dim": 80})
    with pytest.raises(ValueError, match="multiple"):
        QuantDecoderLayer(32, **{**sizes, "heads": 3, "kv_heads": 2})
