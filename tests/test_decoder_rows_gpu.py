"""Rows to int8 on the GPU: RMS norm with residual, rows without a norm, and the training form
with its gradient, against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# half an ulp of a value rounded to the type, relative
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# widths around the shapes that the kernels choose by, and odd ones
COLS = [1, 7, 64, 511, 512, 513, 1024, 1025, 2048, 4099, 8192, 8200, 16385, 40000, 65536]


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def check_codes(codes, exact):
    """Codes are the rounded exact values, but within 1e-4 of a tie either neighbour: u * (127 / a)
    takes three roundings of fp32, at most 127 * 3 * 2^-24 = 2.3e-5."""
    c, r = codes.cpu().numpy().astype(np.int64), np.rint(exact)
    differ = c != r
    near = np.abs(np.abs(exact - np.floor(exact)) - 0.5) < 1e-4
    assert (np.abs(c - r) <= 1).all() and not (differ & ~near).any()


def make(rows, cols, dtype, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 3).to(dtype).to(cuda)
    r = torch.randn(rows, cols, generator=g).to(dtype).to(cuda)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype).to(cuda)
    return x, r, w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_rms_norm_quantize(cuda, cols, dtype):
    rows = 1 if cols > 20000 else 5
    x, r, w = make(rows, cols, dtype, cols, cuda)
    w32 = w.float() * 1.0009765625
    for weight, res in ((w, r), (w32, None)):
        codes, scales, h = ops.rms_norm_quantize(x, weight, res, eps=1e-5)
        want = (x.float() + r.float()).to(dtype) if res is not None else x
        assert torch.equal(h, want) and h.dtype == dtype and codes.dtype == torch.int8
        exact, scale, _ = O.rms_quantize(f64(want), f64(weight), 1e-5)
        check_codes(codes, exact)
        # the mean's sum: at most 64 additions in a chain of a thread and its tree, halved by the root
        assert np.allclose(f64(scales), scale, rtol=40 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 63, 512, 2050, 9000])
def test_quantize_rows(cuda, cols, dtype):
    x, _, _ = make(7, cols, dtype, cols, cuda)
    codes, scales = ops.quantize_rows(x)
    exact, scale = O.quantize_rows(f64(x))
    check_codes(codes, exact)
    assert np.allclose(f64(scales), scale, rtol=2.0 ** -22, atol=0)


def test_rows_that_are_not_finite_or_tiny(cuda):
    """A NaN or an infinity makes its own row NaN and no other one; rows of zeros and of the
    least magnitudes stay finite."""
    x = torch.randn(8, 300, generator=torch.Generator().manual_seed(3)).to(cuda)
    x[1, 7] = float("nan")
    x[2, 299] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = 0
    x[5] = 1e-44
    x[6] *= 1e30
    w = torch.ones(300, device=cuda)
    for codes, scales in (ops.quantize_rows(x), ops.rms_norm_quantize(x, w)[:2]):
        bad = [1, 2, 3]
        assert torch.isnan(scales[bad]).all() and (codes[bad] == 0).all()
        good = [0, 4, 5, 6, 7]
        assert torch.isfinite(scales[good]).all() and (scales[good] >= 0).all()
        assert (codes[4] == 0).all() and (codes[[0, 7]].abs().amax(-1) == 127).all()
    codes, scales = ops.quantize_rows(x)
    assert codes[6].abs().max() == 127
    y, h = ops.rms_norm_quantize_dequantize(x, w)
    assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4, 5, 7]]).all()
    assert torch.equal(torch.nan_to_num(h), torch.nan_to_num(x))


def test_row_views(cuda):
    """Strided rows, more axes, no rows, rows that are a column of something."""
    big = torch.randn(6, 700, generator=torch.Generator().manual_seed(5)).to(cuda).bfloat16()
    w = torch.rand(300, device=cuda).bfloat16() + 0.5
    view = big[::2, 11:311]
    a = ops.rms_norm_quantize(view, w, view)
    b = ops.rms_norm_quantize(view.contiguous(), w, view.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    turned = big.t()[:300]  # a dense first axis
    a, b = ops.quantize_rows(turned), ops.quantize_rows(turned.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c3 = ops.rms_norm_quantize(view.reshape(3, 1, 300), w)
    assert c3[0].shape == (3, 1, 300) and c3[1].shape == (3, 1)
    none = ops.rms_norm_quantize(view[:0], w, view[:0])
    assert none[0].shape == (0, 300) and none[1].shape == (0,)
    spread = ops.quantize_rows(big[:1, :300].expand(4, 300))
    assert all(torch.equal(spread[0][k], spread[0][0]) for k in range(4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 65, 513, 2051, 4096, 8200, 20001])
def test_training_form(cuda, cols, dtype):
    """y is codes * scale of the serving form; gradients against the formula in 64 bits."""
    rows = 1500 if cols == 65 else 9  # more rows than the backward has blocks, and fewer
    x, r, w = make(rows, cols, dtype, cols + 1, cuda)
    g = torch.Generator().manual_seed(cols + 2)
    dy = torch.randn(rows, cols, generator=g).to(dtype).to(cuda)
    dh = torch.randn(rows, cols, generator=g).to(dtype).to(cuda)
    eps = 1e-6
    for res, weight in ((r, w), (None, w.float())):
        leaves = [t.clone().requires_grad_() for t in (x, weight)]
        rl = res.clone().requires_grad_() if res is not None else None
        y, h = ops.rms_norm_quantize_dequantize(leaves[0], leaves[1], rl, eps=eps)
        codes, scales, h2 = ops.rms_norm_quantize(x, weight, res, eps=eps)
        assert torch.equal(h, h2) and torch.equal(y, (codes * scales[:, None]).to(dtype))
        torch.autograd.backward([y, h], [dy, dh])
        dx, dw = O.rms_backward(f64(h2), f64(weight), eps, f64(dy), f64(dh))
        # dx: the row's dot of at most 128 terms a thread, then half an ulp of the type; its terms
        # are at most rstd * |dn| + |n| * mean + |dh|
        rstd = 1 / np.sqrt((f64(h2) ** 2).mean(-1, keepdims=True) + eps)
        dn = np.abs(f64(dy) * f64(weight))
        n = np.abs(f64(h2)) * rstd
        size = rstd * (dn + n * (dn * n).mean(-1, keepdims=True)) + np.abs(f64(dh))
        off = np.abs(f64(leaves[0].grad) - dx)
        assert (off <= HALF_ULP[dtype] * np.abs(dx) + 150 * 2.0 ** -24 * size + 1e-7).all()
        if rl is not None:
            assert torch.equal(rl.grad, leaves[0].grad)
        # dw: rows summed one after the other in a block, then the blocks: at most 200 in a chain
        wsize = np.abs(f64(dy) * f64(h2) * rstd).sum(0)
        half = HALF_ULP[weight.dtype]
        assert (np.abs(f64(leaves[1].grad) - dw) <= half * np.abs(dw) + 200 * 2.0 ** -24 * wsize
                + 1e-7).all()


def test_gradient_against_differences(cuda):
    """Central differences of the smooth norm in 64 bits, in a random direction of each input: the
    step's third-order term is below 1e-7 of the value, fp32's sums below 1e-4."""
    rng = np.random.default_rng(0)
    h, w = rng.standard_normal((4, 200)), 1 + 0.2 * rng.standard_normal(200)
    dy = rng.standard_normal((4, 200))
    h32, w32, dy32 = (torch.tensor(v, dtype=torch.float32, device=cuda) for v in (h, w, dy))
    h32.requires_grad_()
    w32.requires_grad_()
    y, _ = ops.rms_norm_quantize_dequantize(h32, w32, eps=1e-5)
    y.backward(dy32)
    h, w, dy = f64(h32), f64(w32), f64(dy32)
    for k in range(3):
        dir_h, dir_w = rng.standard_normal(h.shape), rng.standard_normal(w.shape)
        t = 1e-4
        up = (O.rms_smooth(h + t * dir_h, w, 1e-5) * dy).sum()
        dn = (O.rms_smooth(h - t * dir_h, w, 1e-5) * dy).sum()
        assert abs((up - dn) / (2 * t) - (f64(h32.grad) * dir_h).sum()) < 2e-3
        up = (O.rms_smooth(h, w + t * dir_w, 1e-5) * dy).sum()
        dn = (O.rms_smooth(h, w - t * dir_w, 1e-5) * dy).sum()
        assert abs((up - dn) / (2 * t) - (f64(w32.grad) * dir_w).sum()) < 2e-3


def test_gradients_that_do_not_arrive(cuda):
    """Only y, or only h, carries a gradient; a weight that needs none gets none; strided and
    broadcast gradients."""
    x, r, w = make(5, 100, torch.float32, 9, cuda)
    x.requires_grad_()
    y, h = ops.rms_norm_quantize_dequantize(x, w, r)
    (gx,) = torch.autograd.grad(h.sum(), x, retain_graph=True)
    assert torch.equal(gx, torch.ones_like(gx))
    (gx,) = torch.autograd.grad(y.sum(), x)  # a gradient of stride 0
    dx, _ = O.rms_backward(f64(x + r), f64(w), 1e-6, np.ones((5, 100)), None)
    assert np.allclose(f64(gx), dx, rtol=0, atol=2e-5)
    assert w.grad is None


def test_more_rows_than_a_launch_takes(cuda):
    """Rows beyond the 2^21 of one launch; the last ones as a call of their own gives them."""
    rows = (1 << 21) + 37
    x = torch.randn(rows, 8, generator=torch.Generator().manual_seed(1)).half().to(cuda)
    codes, scales = ops.quantize_rows(x)
    tail, tail_scales = ops.quantize_rows(x[-40:])
    assert torch.equal(codes[-40:], tail) and torch.equal(scales[-40:], tail_scales)
    exact, _ = O.quantize_rows(f64(x[:50]))
    check_codes(codes[:50], exact)


def test_side_stream_and_same_bits(cuda):
    """Tensors made on another stream than the call's; the same bits on every run."""
    x, r, w = make(64, 4099, torch.bfloat16, 11, cuda)
    first = ops.rms_norm_quantize(x, w, r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.rms_norm_quantize(x, w, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals(cuda):
    x = torch.zeros(2, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ops.rms_norm_quantize(x.cpu(), w)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.quantize_rows(x.double())
    with pytest.raises(RuntimeError, match="needs a weight"):
        ops.rms_norm_quantize(x, None)
    with pytest.raises(RuntimeError, match="shape"):
        ops.rms_norm_quantize(x, w[:7])
    with pytest.raises(RuntimeError, match="weight must be"):
        ops.rms_norm_quantize(x, w.half())
    with pytest.raises(RuntimeError, match="residual"):
        ops.rms_norm_quantize(x, w, x[:1])
    with pytest.raises(RuntimeError, match="rows of 1 to"):
        ops.quantize_rows(torch.zeros(1, 65537, device=cuda))
