"""int8 product with its epilogue on the GPU, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.to(torch.float64).cpu().numpy()


def make(M, N, K, seed, cuda):
    rng = np.random.default_rng(seed)
    x = torch.tensor(rng.integers(-127, 128, (M, K)), dtype=torch.int8, device=cuda)
    w = torch.tensor(rng.integers(-127, 128, (N, K)), dtype=torch.int8, device=cuda)
    sx = torch.tensor(rng.uniform(0.5, 1.5, M) / 127, dtype=torch.float32, device=cuda)
    sw = torch.tensor(rng.uniform(0.5, 1.5, N) / (127 * np.sqrt(K)), dtype=torch.float32, device=cuda)
    return x, sx, w, sw


def check(y, x, sx, w, sw, bias=None, act=None, residual=None):
    want, size = O.linear(x.cpu().numpy(), f64(sx), w.cpu().numpy(), f64(sw),
                          None if bias is None else f64(bias), act,
                          None if residual is None else f64(residual))
    # int32 -> fp32, two products, the bias, the activation (its slope is at most 1.13, its
    # functions within 4 ulp) and the residual: at most 12 half ulps of what was added up
    off = np.abs(f64(y) - want)
    assert (off <= HALF_ULP[y.dtype] * np.abs(want) + 12 * 2.0 ** -24 * size + 1e-7).all(), off.max()


# from one row through the limits of the forms for few rows to whole and ragged tiles
@pytest.mark.parametrize("M", [1, 15, 16, 17, 33, 64, 65, 128, 200, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (130, 100), (257, 1025), (300, 4096)])
def test_sizes(cuda, M, N, K):
    x, sx, w, sw = make(M, N, K, M * 7 + N, cuda)
    check(ops.linear_int8(x, sx, w, sw, dtype=torch.float32), x, sx, w, sw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(5, 70, 96), (150, 259, 320), (513, 512, 256)])
def test_epilogue(cuda, M, N, K, act, dtype):
    x, sx, w, sw = make(M, N, K, 3, cuda)
    g = torch.Generator().manual_seed(4)
    bias = torch.randn(N, generator=g).to(dtype).to(cuda)
    res = torch.randn(M, N, generator=g).to(dtype).to(cuda)
    for b in (None, bias):
        for r in (None, res):
            y = ops.linear_int8(x, sx, w, sw, bias=b, activation=act, residual=r, dtype=dtype)
            assert y.dtype == dtype
            check(y, x, sx, w, sw, b, act, r)


# every shape of tile: whole ones, ragged edges, K that ends inside a step, fewer steps than are
# loaded ahead, K in parts
@pytest.mark.parametrize("M,N,K", [(512, 512, 1024), (700, 1000, 640), (256, 768, 4112), (2049, 513, 192),
                                   (3900, 4100, 208), (4096, 4096, 64), (4096, 4096, 16), (4000, 4099, 130),
                                   (2000, 4100, 336), (1000, 4100, 1040), (1001, 4100, 70), (500, 4096, 272),
                                   (24, 2000, 4112), (60, 1000, 8208), (100, 700, 5000), (90, 500, 4107)])
def test_larger_tiles(cuda, M, N, K):
    x, sx, w, sw = make(M, N, K, 9, cuda)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(cuda)
    check(ops.linear_int8(x, sx, w, sw, bias=bias, dtype=torch.float32), x, sx, w, sw, bias)


@pytest.mark.parametrize("M", [3, 300])
def test_longest_contraction_is_exact(cuda, M):
    """All codes -128, K = 131071: the sum 2^14 * K is the largest that int32 holds here."""
    K = ops.LINEAR_K_MAX
    x = torch.full((M, K), -128, dtype=torch.int8, device=cuda)
    w = torch.full((32, K), -128, dtype=torch.int8, device=cuda)
    one = lambda n: torch.ones(n, device=cuda)
    y = ops.linear_int8(x, one(M), w, one(32), dtype=torch.float32)
    assert (y == float(np.float32(2 ** 14 * K))).all()


@pytest.mark.parametrize("M", [9, 200])
@pytest.mark.parametrize("offset", [0, 1, 16])
def test_strides_and_alignment(cuda, M, offset):
    """Rows of wider tensors, at any byte; a residual of a wider tensor; more axes; no rows."""
    K, N = 160, 130
    x, sx, w, sw = make(M, N, 400, 5, cuda)
    xv, wv = x[:, offset:offset + K], w[:, offset:offset + K]
    res = torch.randn(M, N + 50, generator=torch.Generator().manual_seed(2)).to(cuda)[:, 7:7 + N]
    y = ops.linear_int8(xv, sx, wv, sw, residual=res, dtype=torch.float32)
    check(y, xv, sx, wv, sw, residual=res)
    y3 = ops.linear_int8(xv.reshape(1, M, K), sx.reshape(1, M), wv, sw,
                         residual=res.reshape(1, M, N), dtype=torch.float32)
    assert torch.equal(y3[0], y)
    none = ops.linear_int8(xv[:0], sx[:0], wv, sw)
    assert none.shape == (0, N)
    assert torch.equal(ops.linear_int8(xv, sx[::1], wv.t().contiguous().t(), sw, residual=res,
                                       dtype=torch.float32), y)


@pytest.mark.parametrize("M", [4, 130])
def test_nan_scales_stay_in_their_rows(cuda, M):
    x, sx, w, sw = make(M, 40, 64, 6, cuda)
    sx[2], sw[5] = float("nan"), float("inf")
    y = ops.linear_int8(x, sx, w, sw, dtype=torch.float32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[2], bad[:, 5] = True, True
    assert torch.isfinite(y[~bad]).all() and torch.isnan(y[2]).all()


def test_refusals(cuda):
    x, sx, w, sw = make(4, 8, 16, 1, cuda)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ops.linear_int8(x.cpu(), sx, w, sw)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.linear_int8(x, sx, w, sw, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="activation"):
        ops.linear_int8(x, sx, w, sw, activation="tanh")
    with pytest.raises(RuntimeError, match="codes"):
        ops.linear_int8(x[:, :8], sx, w, sw)
    with pytest.raises(RuntimeError, match="codes"):
        ops.linear_int8(x.float(), sx, w, sw)
    with pytest.raises(RuntimeError, match="scales"):
        ops.linear_int8(x, sx[:3], w, sw)
    with pytest.raises(RuntimeError, match="weight_scales"):
        ops.linear_int8(x, sx, w, sw.double())
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear_int8(x, sx, w, sw, bias=sw, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="residual"):
        ops.linear_int8(x, sx, w, sw, residual=torch.zeros(4, 9, device=cuda), dtype=torch.float32)
    with pytest.raises(RuntimeError, match="columns"):
        ops.linear_int8(torch.zeros(1, 131072, dtype=torch.int8, device=cuda), sx[:1],
                        torch.zeros(1, 131072, dtype=torch.int8, device=cuda), sw[:1])
