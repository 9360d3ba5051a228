"""RMS norm of rows whose squares leave fp32's range, forward and backward, against the definitions in
64 bits."""
import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def make(cols, size, dtype, cuda):
    """Ordinary rows around one of the size and one that has it in a single element."""
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(5, cols, generator=g)
    x[1] *= size
    x[3, cols // 2] = size
    w = 1 + 0.2 * torch.randn(cols, generator=g)
    return x.to(dtype).to(cuda), w.to(cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 300, 1000, 1025, 4099, 8192, 9000, 20001, 65536])
@pytest.mark.parametrize("size,eps", [(3e17, 1e-6), (1e19, 1e-6), (1e25, 1e-6), (1e37, 1e-6), (1e-25, 0.0),
                                      (1e-30, 0.0)])
def test_forward(cuda, cols, dtype, size, eps):
    x, w = make(cols, size, dtype, cuda)
    r = (x.float() * 0.25).to(dtype)
    for res in (None, r):
        codes, scales, h = ops.rms_norm_quantize(x, w, res, eps=eps)
        assert torch.equal(h, x if res is None else (x.float() + r.float()).to(dtype))
        exact, scale, _ = O.rms_quantize(f64(h), f64(w), eps)
        differ = np.abs(codes.cpu().numpy() - exact)
        assert differ.max() <= 0.5001
        # the mean's sum in fp32 of ordinary rows: at most 64 additions in a chain and their tree, halved
        assert np.allclose(f64(scales), scale, rtol=40 * 2.0 ** -24, atol=0)
        y, _ = ops.rms_norm_quantize_dequantize(x, w, res, eps=eps)
        assert torch.equal(y, (codes * scales[:, None]).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [300, 4099, 20001])
@pytest.mark.parametrize("size", [1e19, 1e25, 1e33])
def test_backward(cuda, cols, dtype, size):
    """dx is in units of 1 / size there: its tolerance is relative to its own row."""
    x, w = make(cols, size, dtype, cuda)
    w = w.to(dtype)
    dy = torch.randn(5, cols, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = ops.rms_norm_quantize_dequantize(xl, wl)
    y.backward(dy)
    h, wd, d = f64(x), f64(w), f64(dy)
    dx, dw = O.rms_backward(h, wd, 1e-6, d, None)
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6)
    dn, n = np.abs(d * wd), np.abs(h) * rstd
    size_dx = rstd * (dn + n * (dn * n).mean(-1, keepdims=True))
    tol = HALF_ULP[dtype] * np.abs(dx) + 150 * 2.0 ** -24 * size_dx
    assert (np.abs(f64(xl.grad) - dx) <= tol).all()
    tol = HALF_ULP[dtype] * np.abs(dw) + 200 * 2.0 ** -24 * (np.abs(d) * n).sum(0)
    assert (np.abs(f64(wl.grad) - dw) <= tol).all()


def test_rows_that_are_not_finite(cuda):
    """They stay NaN beside rows beyond the range of squares; a product with the weight beyond fp32 is
    an infinity."""
    x = torch.ones(4, 600, device=cuda) * 1e20
    x[0, 3], x[1, 5] = float("inf"), float("nan")
    codes, scales, _ = ops.rms_norm_quantize(x, torch.ones(600, device=cuda))
    assert torch.isnan(scales[:2]).all() and (codes[:2] == 0).all()
    assert np.allclose(f64(scales[2:]), 1 / 127, rtol=1e-6) and (codes[2:] == 127).all()
    scales = ops.rms_norm_quantize(x, torch.full((600,), 1e20, device=cuda))[1]
    assert torch.isnan(scales).all()
