"""NaNs of any sign and payload: their row or page has scale NaN and codes 0."""
import numpy as np
import pytest
import torch

import decoder_ops as ops

pytestmark = pytest.mark.gpu

PAYLOADS = np.array([0x7fc00001, 0x7f800080, 0xffc000ff, 0x7fffffff], np.uint32)


def nans(cuda, rows, cols):
    """Every row has one of the NaNs, and ordinary values beside it."""
    x = np.random.default_rng(0).standard_normal((rows, cols)).astype(np.float32)
    x.view(np.uint32)[np.arange(rows), 3] = np.resize(PAYLOADS, rows)
    return torch.from_numpy(x).to(cuda)


def test_rows(cuda):
    for cols in (9, 600, 3000):
        x = nans(cuda, 4, cols)
        for codes, scales in (ops.quantize_rows(x), ops.rms_norm_quantize(x, torch.ones(cols, device=cuda))[:2]):
            assert torch.isnan(scales).all() and (codes == 0).all()


def test_cache(cuda):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    cache = ops.KVCache.empty(4, 1, 64, 16, device=cuda)
    for t in cache:
        t.fill_(1)
    x = nans(cuda, 4, 64)[:, None]
    ops.kv_cache_append(cache, x, x, ints(0, 1, 2, 3)[:, None], ints(0, 0, 0, 0))
    assert torch.isnan(cache.k_scale).all() and torch.isnan(cache.v_scale).all()
    assert (cache.k[:, :, 0] == 0).all() and (cache.v[..., 0] == 0).all()
