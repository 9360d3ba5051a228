"""Products whose scales lie at the ends of fp32 while their results do not, against the definition in
64 bits: few rows, tiles, and K in parts."""
import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(3, 70, 200), (40, 70, 4096), (200, 130, 200)])
@pytest.mark.parametrize("sx,sw", [(1e35, 1e-36), (1e-36, 1e35), (2e36, 1e-30), (-1e35, 1e-36), (1e-30, 1e-9)])
def test_scales_at_the_ends_of_the_range(cuda, M, N, K, sx, sw):
    g = torch.Generator().manual_seed(0)
    x = torch.randint(60, 128, (M, K), generator=g).to(torch.int8).to(cuda)  # of one sign: nothing cancels
    w = torch.randint(60, 128, (N, K), generator=g).to(torch.int8).to(cuda)
    ax = (1 + torch.rand(M, generator=g)).to(cuda) * sx
    ax[1] = 0.5  # an ordinary row beside the others
    aw = (1 + torch.rand(N, generator=g)).to(cuda) * sw
    y = ops.linear_int8(x, ax, w, aw, dtype=torch.float32).double().cpu().numpy()
    f = lambda t: t.double().cpu().numpy()
    want, _ = O.linear(x.cpu().numpy(), f(ax), w.cpu().numpy(), f(aw), None, None, None)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)  # the ordinary row is beyond it where weight scales are large
    # the sum rounded to fp32, two products
    assert np.allclose(y, want, rtol=4 * 2.0 ** -24, atol=2.0 ** -126)
