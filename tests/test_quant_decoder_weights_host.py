"""Feed-forward weights that a layer made from float weights cannot use are refused, not dropped."""
import pytest
import torch

from quant_decoder import QuantDecoderLayer, QuantExperts


@pytest.mark.parametrize("up,down,with_experts", [(True, False, False), (False, True, False), (True, False, True),
                                                  (False, True, True), (True, True, True)])
def test_both_products_or_neither(up, down, with_experts):
    experts = QuantExperts(64, 48, 8, 2, device="cpu") if with_experts else None
    with pytest.raises(ValueError, match="w_up and w_down"):
        QuantDecoderLayer.from_float(
            torch.ones(64), torch.ones(256, 64), torch.ones(64, 128), torch.ones(64),
            torch.ones(48, 64) if up else None, torch.ones(64, 48) if down else None,
            heads=2, kv_heads=1, experts=experts)


def test_neither_products_nor_experts():
    with pytest.raises(ValueError, match="either hidden or experts"):
        QuantDecoderLayer.from_float(torch.ones(64), torch.ones(256, 64), torch.ones(64, 128), torch.ones(64),
                                     heads=2, kv_heads=1)
