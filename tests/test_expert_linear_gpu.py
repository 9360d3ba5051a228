"""int8 product with a weight for each expert on the GPU, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def make(T, k, E, N, K, seed, cuda, gated=False, grouped=False, share_out=0.0, ids=None):
    rng = np.random.default_rng(seed)
    if ids is None:
        ids = rng.integers(0, E, (T, k)).astype(np.int32)
        ids[rng.random((T, k)) < share_out] = -1
    g = ops.group_experts(torch.tensor(ids, dtype=torch.int32, device=cuda), E)
    rows, out = T * k if grouped else T, N * (1 + gated)
    t = lambda a, d: torch.tensor(a, dtype=d, device=cuda)
    x = t(rng.integers(-127, 128, (rows, K)), torch.int8)
    w = t(rng.integers(-127, 128, (E, out, K)), torch.int8)
    sx = t(rng.uniform(0.5, 1.5, rows) / 127, torch.float32)
    sw = t(rng.uniform(0.5, 1.5, (E, out)) / (127 * np.sqrt(K)), torch.float32)
    b = t(rng.standard_normal((E, out)), torch.float32)
    return x, sx, w, sw, g, b


def check(x, sx, w, sw, g, bias=None, act=None, gated=False, grouped=False, dtype=torch.float32):
    y = ops.experts_linear_int8(x, sx, w, sw, g, bias=bias, activation=act, gated=gated, grouped=grouped,
                                dtype=dtype)
    k = g.places.shape[-1]
    assert y.dtype == dtype and y.shape == (g.places.numel(), w.shape[1] // (1 + gated))
    want, size = O.linear(x.cpu().numpy(), f64(sx), w.cpu().numpy(), f64(sw), g.offsets.cpu().numpy(),
                          g.entries.cpu().numpy(), k, None if bias is None else f64(bias), act, gated, grouped)
    off = np.abs(f64(y[:len(want)]) - want)
    # int32 -> fp32, two products, the bias and the activation (its slope is at most 1.13, its functions
    # within 4 ulp): at most 12 half steps of what was added up; where gated, both factors and their product
    bound = HALF_STEP[dtype] * np.abs(want) + 26 * 2.0 ** -24 * size + 1e-7
    assert (off <= bound).all(), (off / bound).max()
    return y


# from one row to several tiles of an expert, through the limits of each form; widths and depths that are odd
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 2, 8), (16, 8, 64), (31, 1, 2), (40, 3, 5), (300, 1, 3),
                                   (100, 4, 3), (700, 2, 4), (600, 1, 1), (1500, 2, 3)])
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (130, 100), (67, 1025), (300, 512)])
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(cuda, T, k, E, N, K, gated):
    x, sx, w, sw, g, b = make(T, k, E, N, K, T + N, cuda, gated)
    check(x, sx, w, sw, g, b, "silu" if gated else None, gated)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("T", [20, 700, 2000])
@pytest.mark.parametrize("gated,grouped", [(False, True), (True, False), (True, True)])
def test_epilogue(cuda, dtype, act, T, gated, grouped):
    x, sx, w, sw, g, b = make(T, 2, 4, 72, 128, T, cuda, gated, grouped, share_out=0.2)
    check(x, sx, w, sw, g, b.to(dtype), act, gated, grouped, dtype)
    check(x, sx, w, sw, g, None, act, gated, grouped, dtype)


@pytest.mark.parametrize("T", [30, 600, 2500])
@pytest.mark.parametrize("K", [64, 96, 1000])
def test_uneven_experts(cuda, T, K):
    for ids in (np.zeros((T, 2), np.int32), np.full((T, 2), -1, np.int32), np.full((T, 2), 5, np.int32),
                np.stack([np.arange(T) % 3, np.full(T, 4)], 1)):
        x, sx, w, sw, g, b = make(T, 2, 6, 80, K, 3, cuda, ids=ids)
        check(x, sx, w, sw, g, b)


@pytest.mark.parametrize("T", [8, 500])
def test_rows_of_no_expert_are_not_written(cuda, T):
    x, sx, w, sw, g, _ = make(T, 2, 3, 40, 64, 4, cuda, share_out=0.5)
    held = int(g.offsets[-1])
    marks = torch.full((T * 2, 40), 7.0, device=cuda)
    at = marks.data_ptr()
    del marks  # the allocator hands the same memory out again
    y = ops.experts_linear_int8(x, sx, w, sw, g, dtype=torch.float32)
    if y.data_ptr() == at:
        assert (y[held:] == 7).all()


@pytest.mark.parametrize("T", [12, 900])
def test_nan_infinite_and_large_scales(cuda, T):
    x, sx, w, sw, g, _ = make(T, 2, 3, 48, 64, 5, cuda)
    sx[0], sx[1], x[1] = torch.nan, torch.inf, 0
    x[2], sx[2] = 127, 2.0 ** 120       # the row's scale alone would leave fp32
    sw *= 2.0 ** -110
    y = ops.experts_linear_int8(x, sx, w, sw, g, dtype=torch.float32)
    places = g.places
    assert y[places[0].long()].isnan().all() and y[places[1].long()].isnan().all()
    want = x[2].double() @ w.double().transpose(1, 2) * sx[2].double() * sw.double()
    e = torch.searchsorted(g.offsets[1:].contiguous(), places[2], right=True)
    assert torch.allclose(y[places[2].long()].double(), want[e], rtol=1e-6)


@pytest.mark.parametrize("T", [10, 400, 1600])
def test_strides_and_alignment(cuda, T):
    x, sx, w, sw, g, b = make(T, 2, 3, 50, 200, 6, cuda)
    for off, K in ((0, 128), (16, 128), (1, 128), (3, 77), (16, 100)):
        xs, ws = x[:, off:off + K], w[:, :, off:off + K]
        want = ops.experts_linear_int8(xs.contiguous(), sx, ws.contiguous(), sw, g, dtype=torch.float32)
        assert torch.equal(ops.experts_linear_int8(xs, sx, ws, sw, g, dtype=torch.float32), want)
    every = w.repeat(1, 2, 1)[:, ::2]  # rows, then experts, that are not side by side
    s2 = sw.repeat(1, 2)[:, ::2]
    want = ops.experts_linear_int8(x, sx, every.contiguous(), s2.contiguous(), g, dtype=torch.float32)
    assert torch.equal(ops.experts_linear_int8(x, sx, every, s2, g, dtype=torch.float32), want)
    turned = w.transpose(1, 2).contiguous().transpose(1, 2)  # a last axis that is not dense
    want = ops.experts_linear_int8(x, sx, w, sw, g, dtype=torch.float32)
    assert torch.equal(ops.experts_linear_int8(x, sx, turned, sw, g, dtype=torch.float32), want)
    same = w[:1].expand(3, -1, -1)     # one weight for all
    want = ops.experts_linear_int8(x, sx, same.contiguous(), sw, g, dtype=torch.float32)
    assert torch.equal(ops.experts_linear_int8(x, sx, same, sw, g, dtype=torch.float32), want)


@pytest.mark.parametrize("T", [8, 300, 2000])
def test_groups_out_of_range_stay_in_bounds(cuda, T):
    """Offsets and entries that no order of the tokens has: rows of no expert, or of the nearest token."""
    x, sx, w, sw, g, _ = make(T, 2, 3, 48, 64, 7, cuda)
    n = 2 * T
    run = lambda offsets, entries=g.entries: ops.experts_linear_int8(
        x, sx, w, sw, ops.ExpertGroups(torch.tensor(offsets, dtype=torch.int32, device=cuda), entries, g.places),
        dtype=torch.float32)
    run([-5, 4, n + 100, 2 ** 31 - 1])
    run([n, 0, n, 0])
    run([0, n, -2 ** 31, n])
    far = g.entries.clone()
    far[0], far[1], far[-1] = -1, -2 ** 31, 2 ** 31 - 1
    near = g.entries.clone()
    near[0], near[1], near[-1] = 0, 0, n - 1
    at = g.offsets.tolist()
    assert torch.equal(run(at, far), run(at, near))
    torch.cuda.synchronize()


def test_no_tokens(cuda):
    x, sx, w, sw, g, _ = make(0, 2, 3, 48, 64, 8, cuda)
    assert ops.experts_linear_int8(x, sx, w, sw, g).shape == (0, 48)


def test_refusals(cuda):
    x, sx, w, sw, g, b = make(6, 2, 3, 16, 32, 9, cuda)
    call = lambda **kw: ops.experts_linear_int8(**{**dict(codes=x, scales=sx, weight=w, weight_scales=sw,
                                                          groups=g, dtype=torch.float32), **kw})
    call()
    for kw, match in ((dict(codes=x[:5]), "codes must have"), (dict(codes=x.float()), "codes must be"),
                      (dict(grouped=True), "codes must have"), (dict(scales=sx[:5]), "scales must have"),
                      (dict(scales=sx.double()), "scales must be"), (dict(weight=w[:2]), "experts of groups"),
                      (dict(weight=w[:, :, 1:]), "codes must have"), (dict(weight=w.float()), "weight must be"),
                      (dict(weight_scales=sw[:, 1:]), "weight_scales must have"),
                      (dict(bias=b[:, 1:]), "bias must have"), (dict(bias=b.half()), "bias must be"),
                      (dict(activation="tanh"), "activation"), (dict(dtype=torch.float64), "dtype"),
                      (dict(weight=w[:, 1:], weight_scales=sw[:, 1:], gated=True), "even number"),
                      (dict(codes=x[0]), "codes must be"), (dict(weight=w.cpu()), "weight must be")):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
