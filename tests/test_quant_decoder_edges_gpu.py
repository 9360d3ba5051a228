"""A decoder layer on passes without tokens."""
import pytest
import torch

from quant_decoder import KVCache, QuantDecoderLayer, Step

pytestmark = pytest.mark.gpu


def test_a_pass_without_tokens(cuda):
    """No rows, for no sequence and for sequences that bring none: no rows out, the cache as it was."""
    layer = QuantDecoderLayer(128, heads=2, kv_heads=1, head_dim=64, hidden=128, device=cuda)
    cache = KVCache.empty(2, 1, 64, 16, device=cuda)
    for t in cache:
        t.fill_(3)
    x = torch.empty(0, 128, dtype=torch.bfloat16, device=cuda)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    for step in (Step(ints(0, 1).view(2, 1), ints(5, 0), ints(0, 0, 0), 0, 16),
                 Step(torch.empty(0, 1, dtype=torch.int32, device=cuda), ints(), None, None, 16)):
        y = layer(x, cache, step)
        assert y.shape == (0, 128) and y.dtype == torch.bfloat16
    assert all((t == 3).all() for t in cache)
