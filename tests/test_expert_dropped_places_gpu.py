"""Rows that belong to no entry: gradients of places that a caller takes away (what exceeds an expert's
capacity), and the product's rows behind the experts' last place."""
import ctypes

import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O
import rxmet_lib

pytestmark = pytest.mark.gpu


def make(cuda, T, k, N, E, dtype, seed):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < 0.1] = -1
    g = ops.group_experts(torch.tensor(ids, device=cuda), E)
    t = lambda *s: torch.tensor(rng.standard_normal(s), dtype=torch.float32, device=cuda)
    drop = torch.tensor(rng.random((T, k)) < 0.3, device=cuda)
    places = torch.where(drop, -1, g.places)
    places[T // 2] = -1  # a token of which nothing is left
    return t(T * k, N).to(dtype), t(T, k), ops.ExpertGroups(g.offsets, g.entries, places), t(T, N).to(dtype)


def named(g):
    """Which rows a place names."""
    rows = torch.zeros(g.places.numel(), dtype=torch.bool, device=g.places.device)
    rows[g.places[g.places >= 0].long()] = True
    return rows


@pytest.mark.parametrize("T,k,N", [(1, 3, 5), (40, 2, 33), (30, 8, 1000), (25, 10, 4100), (1024, 4, 70), (1366, 3, 33),
                                   (4100, 2, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_rows_without_an_entry_is_zero(cuda, T, k, N, dtype):
    y, w, g, d = make(cuda, T, k, N, 4, dtype, T + N)
    # the library itself, on a gradient that holds something else before
    dy = torch.full_like(y, 7.0)
    dw = torch.full_like(w, 7.0)
    at = rxmet_lib.ExpertGroups(*(t.data_ptr() for t in g), T, k, 4)
    rxmet_lib.call("rxmet_experts_combine_backward", ctypes.byref(at), d.data_ptr(), N, y.data_ptr(), N,
                   w.data_ptr(), dy.data_ptr(), dw.data_ptr(), N, ops._DTYPE[dtype], rxmet_lib.stream_of(cuda))
    rows = named(g)
    assert int((~rows).sum()) > 0 and (dy[~rows] == 0).all()
    f64 = lambda t: t.double().cpu().numpy()
    want, dw64, size = O.combine_backward(f64(y), f64(w), g.places.cpu().numpy(), f64(d))
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    # one product in fp32, rounded to y's type; sums of N products
    assert (np.abs(f64(dy) - want) <= (half + 2.0 ** -24) * 1.01 * np.abs(want) + tiny).all()
    assert (np.abs(f64(dw) - dw64) <= (N + 8) * 2.0 ** -24 * 1.01 * size).all()
    # and the same through the operator
    y.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(ops.experts_combine(y, w, g), (y, w), d)
    assert torch.equal(got[0], dy) and torch.equal(got[1], dw)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("T", [60, 1200])
def test_places_of_another_order(cuda, monkeypatch, native, T):
    """Places that `entries` does not know: the sum and its gradient go by the places alone."""
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    y, w, g, d = make(cuda, T, 4, 50, 5, torch.float32, 9)
    order = torch.randperm(4 * T, device=cuda, generator=torch.Generator(cuda).manual_seed(1)).int()
    places = torch.where(g.places < 0, -1, order.view(T, 4))
    other = ops.ExpertGroups(g.offsets, g.entries, places)
    y.requires_grad_(), w.requires_grad_()
    out = ops.experts_combine(y, w, other)
    dy, dw = torch.autograd.grad(out, (y, w), d)
    f64 = lambda t: t.detach().double().cpu().numpy()
    p = places.cpu().numpy()
    want, size = O.combine(f64(y), f64(w), p, None)
    # four fused products and sums, one rounding each; one product; sums of 50 products
    assert (np.abs(f64(out) - want) <= 5 * 2.0 ** -24 * 1.01 * size).all()
    dy64, dw64, size = O.combine_backward(f64(y), f64(w), p, f64(d))
    assert (np.abs(f64(dy) - dy64) <= 2.0 ** -24 * 1.01 * np.abs(dy64)).all()
    assert (np.abs(f64(dw) - dw64) <= 58 * 2.0 ** -24 * 1.01 * size).all()


@pytest.mark.parametrize("T", [8, 500])
@pytest.mark.parametrize("K", [64, 100])
def test_product_leaves_rows_of_no_expert_as_they_were(cuda, T, K):
    rng = np.random.default_rng(T)
    ids = rng.integers(0, 3, (T, 2)).astype(np.int32)
    ids[rng.random((T, 2)) < 0.5] = -1
    g = ops.group_experts(torch.tensor(ids, device=cuda), 3)
    held, N = int(g.offsets[-1]), 40
    x = torch.randint(-127, 128, (T, K), dtype=torch.int8, device=cuda)
    w = torch.randint(-127, 128, (3, N, K), dtype=torch.int8, device=cuda)
    sx, sw = torch.rand(T, device=cuda), torch.rand(3, N, device=cuda)
    y = torch.full((2 * T, N), 7.0, device=cuda)
    at = rxmet_lib.ExpertGroups(*(t.data_ptr() for t in g), T, 2, 3)
    rxmet_lib.call("rxmet_experts_linear_int8", ctypes.byref(at), 0, x.data_ptr(), K, sx.data_ptr(), w.data_ptr(), K,
                   N * K, sw.data_ptr(), None, y.data_ptr(), N, K, 0, 0, 0, rxmet_lib.stream_of(cuda))
    assert 0 < held < 2 * T and (y[held:] == 7).all()
    assert torch.equal(y[:held], ops.experts_linear_int8(x, sx, w, sw, g, dtype=torch.float32)[:held])
