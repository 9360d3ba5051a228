"""What a feed-forward of experts and a layer with one refuse when they are made."""
import pytest
import torch

from quant_decoder import QuantDecoderLayer, QuantExperts


def test_experts_that_no_pass_would_take():
    sizes = dict(width=32, hidden=48, experts=8, device="cpu")
    QuantExperts(top_k=2, **sizes)
    for kw, match in ((dict(top_k=9), "top_k"), (dict(top_k=2, score="tanh"), "score"),
                      (dict(top_k=2, groups=3), "groups"), (dict(top_k=2, activation="tanh"), "activation"),
                      (dict(top_k=2, dtype=torch.float64), "dtype")):
        with pytest.raises(ValueError, match=match):
            QuantExperts(**sizes, **kw)


def test_a_layer_has_products_or_experts():
    m = QuantExperts(64, 48, 8, 2, device="cpu")
    layer = QuantDecoderLayer(64, 2, 1, 64, None, experts=m, device="cpu")
    assert "w_up" not in dict(layer.named_buffers()) and layer.experts is m
    with pytest.raises(ValueError, match="either hidden or experts"):
        QuantDecoderLayer(64, 2, 1, 64, None, device="cpu")
    with pytest.raises(ValueError, match="either hidden or experts"):
        QuantDecoderLayer(64, 2, 1, 64, 48, experts=m, device="cpu")
    with pytest.raises(TypeError, match="heads"):
        QuantDecoderLayer.from_float(torch.ones(64), torch.ones(4, 64), torch.ones(64, 4), torch.ones(64))
