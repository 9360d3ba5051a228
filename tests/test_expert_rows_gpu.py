"""The entries' order by expert and the sum of a token's rows on the GPU, against their definitions."""
import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def chosen(T, k, E, seed, share_out=0.1):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < share_out] = -1
    return ids


def check_groups(ids, E, cuda):
    got = ops.group_experts(torch.tensor(ids, device=cuda), E)
    for name, g, w in zip(got._fields, got, O.group(ids, E)):
        assert g.dtype == torch.int32 and tuple(g.shape) == w.shape
        assert np.array_equal(g.cpu().numpy(), w), name
    return got


# one entry, a wave, a chunk, the last size of one launch and the first of two, many chunks
@pytest.mark.parametrize("T,k", [(1, 1), (1, 64), (13, 5), (64, 1), (65, 1), (341, 3), (512, 2), (1024, 4),
                                 (4097, 1), (1366, 3), (5000, 8), (16384, 8)])
@pytest.mark.parametrize("E", [1, 2, 63, 64, 65, 256, 1023, 1024])
def test_order(cuda, T, k, E):
    check_groups(chosen(T, k, E, T + E), E, cuda)


# the last number of chunks that each adds up the others' counts, the first that are added up in between
@pytest.mark.parametrize("n", [128 * 1024, 128 * 1024 + 1, 1500 * 1024 + 77])
@pytest.mark.parametrize("E", [3, 64, 1024])
def test_many_entries(cuda, n, E):
    ids = torch.randint(-1, E + 1, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(n))
    got = ops.group_experts(ids.view(-1, 1).to(cuda), E)
    bins = torch.where((ids < 0) | (ids >= E), E, ids)
    ordered, entries = bins.sort(stable=True)
    places = torch.empty(n, dtype=torch.int32)
    places[entries] = torch.arange(n, dtype=torch.int32)
    places[bins == E] = -1
    assert torch.equal(got.entries.cpu(), entries.int()) and torch.equal(got.places.cpu().view(-1), places)
    assert torch.equal(got.offsets.cpu(), torch.searchsorted(ordered, torch.arange(E + 1, dtype=torch.int32)).int())


@pytest.mark.parametrize("T", [7, 3000])
def test_uneven_choices(cuda, T):
    check_groups(np.zeros((T, 4), np.int32), 9, cuda)              # all to one
    check_groups(np.full((T, 4), -1, np.int32), 9, cuda)           # none
    ids = chosen(T, 4, 9, 1)
    ids[ids == 3] = 200                                            # ids above, an expert without entries
    ids[0, 0] = -2 ** 31
    ids[0, 1] = 2 ** 31 - 1
    check_groups(ids, 9, cuda)
    check_groups(np.arange(T * 4, dtype=np.int32).reshape(T, 4)[::-1] % 9, 9, cuda)


def test_no_entries_leading_axes_and_strides(cuda):
    g = ops.group_experts(torch.empty(0, 3, dtype=torch.int32, device=cuda), 4)
    assert g.offsets.tolist() == [0] * 5 and g.entries.shape == (0,) and g.places.shape == (0, 3)
    ids = torch.tensor(chosen(24, 6, 5, 2), device=cuda)
    want = ops.group_experts(ids[:, 2:4].contiguous(), 5)
    assert all(torch.equal(a, b) for a, b in zip(ops.group_experts(ids[:, 2:4], 5), want))
    got = ops.group_experts(ids[:, 2:4].reshape(2, 3, 4, 2), 5)
    assert got.places.shape == (2, 3, 4, 2) and torch.equal(got.places.view(24, 2), want.places)


def make(T, k, N, E, dtype, seed, cuda, share_out=0.2):
    rng = np.random.default_rng(seed)
    t = lambda *s: torch.tensor(rng.standard_normal(s), dtype=torch.float32, device=cuda)
    g = ops.group_experts(torch.tensor(chosen(T, k, E, seed, share_out), device=cuda), E)
    return t(T * k, N).to(dtype), t(T, k), g, t(T, N).to(dtype)


def check_combine(y, w, g, residual, grad):
    y, w = y.clone(), w.clone()
    held = int(g.offsets[-1])
    with torch.no_grad():
        y[held:] = torch.nan  # rows of no expert are not read
    leaves = [t.requires_grad_() for t in (y, w)] + ([residual.clone().requires_grad_()] if residual is not None else [])
    out = ops.experts_combine(y, w, g, residual=leaves[2] if residual is not None else None)
    places = g.places.cpu().numpy()
    y64 = np.nan_to_num(f64(y))
    want, size = O.combine(y64, f64(w), places, None if residual is None else f64(residual))
    k, half = places.shape[1], HALF_STEP[y.dtype]
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    # one rounding for each row's fused product and sum, one for the residual, one to y's type
    bound = half * np.abs(want) + (k + 2) * 2.0 ** -24 * 1.01 * size + tiny
    assert out.dtype == y.dtype and (np.abs(f64(out) - want) <= bound).all()
    grads = torch.autograd.grad(out, leaves, grad)
    dy, dw, dsize = O.combine_backward(y64, f64(w), places, f64(grad))
    # the product in fp32, rounded again to y's type
    assert (np.abs(f64(grads[0]) - dy) <= (half + 2.0 ** -24 * 1.01) * np.abs(dy) * 1.01 + tiny).all()
    # a sum of N products: none of its partial sums is off by more than N + 8 half steps of their size
    N = y.shape[1]
    assert (np.abs(f64(grads[1]) - dw) <= (N + 8) * 2.0 ** -24 * 1.01 * dsize).all()
    assert (grads[0][held:] == 0).all()
    if residual is not None:
        assert torch.equal(grads[2], grad)
    return out


@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (1, 8, 64), (3, 2, 7), (16, 8, 128), (5, 3, 2048), (9, 5, 2049),
                                   (130, 4, 100), (2, 64, 33), (40, 1, 4099), (3, 6, 9000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_residual", [False, True])
def test_combine_and_its_gradients(cuda, T, k, N, dtype, with_residual):
    y, w, g, r = make(T, k, N, 5, dtype, T + N, cuda)
    grad = torch.randn(T, N, device=cuda, generator=torch.Generator(cuda).manual_seed(N)).to(dtype)
    check_combine(y, w, g, r if with_residual else None, grad)


def test_combine_of_nothing_and_of_strided_rows(cuda):
    y, w, g, r = make(12, 3, 40, 4, torch.bfloat16, 3, cuda, share_out=1.0)
    assert (g.places == -1).all()
    assert torch.equal(ops.experts_combine(y, w, g, residual=r), r)
    assert (ops.experts_combine(y, w, g) == 0).all()
    y, w, g, r = make(12, 3, 50, 4, torch.float16, 4, cuda)
    want = ops.experts_combine(y[:, 3:43].contiguous(), w, g, residual=r[:, 5:45].contiguous())
    assert torch.equal(ops.experts_combine(y[:, 3:43], w, g, residual=r[:, 5:45]), want)
    assert torch.equal(ops.experts_combine(y[:, 3:43].t().contiguous().t(), w.t().contiguous().t(), g,
                                           residual=r[:, 5:45]), want)
    empty = ops.group_experts(torch.empty(0, 3, dtype=torch.int32, device=cuda), 4)
    y0, w0 = y[:0].clone().requires_grad_(), w[:0].clone().requires_grad_()
    out = ops.experts_combine(y0, w0, empty)
    assert out.shape == (0, 50)
    assert [d.shape for d in torch.autograd.grad(out.sum(), (y0, w0))] == [(0, 50), (0, 3)]


@pytest.mark.parametrize("leaf", [0, 1, 2])
def test_gradients_asked_for_one_by_one(cuda, leaf):
    y, w, g, r = make(20, 3, 70, 4, torch.float32, 5, cuda)
    args = [y, w, r]
    args[leaf].requires_grad_()
    grad = torch.randn(20, 70, device=cuda)
    (d,) = torch.autograd.grad(ops.experts_combine(args[0], args[1], g, residual=args[2]), args[leaf], grad)
    all_ = [t.detach().clone().requires_grad_() for t in args]
    want = torch.autograd.grad(ops.experts_combine(all_[0], all_[1], g, residual=all_[2]), all_, grad)[leaf]
    assert torch.equal(d, want)


def test_combine_gradient_against_differences(cuda):
    y, w, g, r = make(8, 3, 33, 4, torch.float32, 6, cuda)
    a, b = torch.randn_like(y), torch.randn_like(w)
    y.requires_grad_(), w.requires_grad_()
    grad = torch.randn(8, 33, device=cuda)
    dy, dw = torch.autograd.grad(ops.experts_combine(y, w, g, residual=r), (y, w), grad)
    f = lambda s: (ops.experts_combine(y.detach() + s * a, w.detach() + s * b, g).double() * grad.double()).sum()
    slope = (f(0.25) - f(-0.25)) / 0.5  # the sum is bilinear: differences are exact up to rounding
    want = (dy.double() * a).sum() + (dw.double() * b).sum()
    assert abs(slope - want) < 1e-4 * (dy.double().norm() * a.double().norm() + dw.double().norm() * b.double().norm())


def test_places_out_of_range_read_nothing(cuda):
    y, w, g, _ = make(6, 2, 16, 3, torch.float32, 7, cuda, share_out=0)
    bad = g.places.clone()
    bad[0, 0], bad[1, 1] = 12, 2 ** 31 - 1
    none = bad.clone()
    none[0, 0] = none[1, 1] = -1
    at = lambda p: ops.ExpertGroups(g.offsets, g.entries, p)
    assert torch.equal(ops.experts_combine(y, w, at(bad)), ops.experts_combine(y, w, at(none)))
    w.requires_grad_()
    d = [torch.autograd.grad(ops.experts_combine(y, w, at(p)).sum(), w)[0] for p in (bad, none)]
    assert torch.equal(*d)


def test_refusals(cuda):
    ids = torch.zeros(4, 2, dtype=torch.int32, device=cuda)
    for what, match in ((lambda: ops.group_experts(ids.long(), 3), "experts must be"),
                        (lambda: ops.group_experts(ids, 0), "1 to 1024"),
                        (lambda: ops.group_experts(ids, 1025), "1 to 1024"),
                        (lambda: ops.group_experts(torch.zeros(2, 65, dtype=torch.int32, device=cuda), 3), "top_k"),
                        (lambda: ops.group_experts(ids[0, 0], 3), "top_k")):
        with pytest.raises(RuntimeError, match=match):
            what()
    y, w, g, r = make(6, 2, 16, 3, torch.float32, 8, cuda)
    for what, match in ((lambda: ops.experts_combine(y[:-1], w, g), "row for each entry"),
                        (lambda: ops.experts_combine(y.double(), w, g), "float32, float16 or bfloat16"),
                        (lambda: ops.experts_combine(y, w.half(), g), "weights must be"),
                        (lambda: ops.experts_combine(y, w[:, :1], g), "weights must have"),
                        (lambda: ops.experts_combine(y, w, g, residual=r.half()), "residual must be"),
                        (lambda: ops.experts_combine(y, w, g, residual=r[:, 1:]), "residual must have"),
                        (lambda: ops.experts_combine(y, w, g._replace(offsets=g.offsets.long())), "offsets"),
                        (lambda: ops.experts_combine(y, w, g._replace(entries=g.entries[1:])), "entries"),
                        (lambda: ops.experts_combine(y, w, g._replace(places=g.places.cpu())), "places")):
        with pytest.raises(RuntimeError, match=match):
            what()
    w.requires_grad_()
    (d,) = torch.autograd.grad(ops.experts_combine(y, w, g).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        d.sum().backward()
