"""Routing to experts on the GPU, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def logits(T, E, seed, cuda, dtype=torch.float32, spread=2.0):
    rng = np.random.default_rng(seed)
    return torch.tensor(rng.standard_normal((T, E)) * spread, dtype=torch.float32, device=cuda).to(dtype)


def check(x, k, bias=None, grad_seed=None, renormalize=True, scale=1.0, **kw):
    """The choice exactly; weights within a rounding of 64 bits to fp32 and the functions' own last bits."""
    x = x.clone().requires_grad_(grad_seed is not None)
    e, w = ops.route_experts(x, k, bias=bias, renormalize=renormalize, scale=scale, **kw)
    choice = dict(kw)
    score = choice.pop("score", "softmax")
    want = O.choose(f64(x), k, score, None if bias is None else bias.cpu().numpy(), **choice)
    assert e.dtype == torch.int32 and w.dtype == torch.float32
    assert np.array_equal(e.cpu().numpy(), want)
    exact = O.weights(f64(x), want, score, renormalize, np.float32(scale))
    # half a step of fp32, some steps of fp64 before it; below its normal range half of the least step
    np.testing.assert_allclose(f64(w), exact, rtol=2.0 ** -24 * 1.001, atol=2.0 ** -150)
    if grad_seed is not None:
        g = torch.tensor(np.random.default_rng(grad_seed).standard_normal(w.shape), dtype=torch.float32,
                         device=x.device)
        (dx,) = torch.autograd.grad(w, x, g)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        want = O.route_backward(f64(x), want, f64(g), score, renormalize, np.float32(scale))
        # rounded to fp32 and to x's type; for softmax as it is p, the difference and their product are fp32
        size = np.abs(f64(g)).sum(-1, keepdims=True) * abs(scale)
        half = torch.finfo(x.dtype).eps / 2
        tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        bound = half * np.abs(want) + 16 * 2.0 ** -24 * size * np.minimum(1, O.scores(f64(x), score)) + tiny
        off = np.abs(f64(dx) - want)
        assert (off <= bound).all(), (off / bound).max()
    return e, w


# one token, odd numbers of experts, the limits of each number of lanes
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 7, 7), (5, 60, 4), (16, 64, 8), (17, 65, 6),
                                   (33, 128, 3), (9, 160, 6), (50, 256, 8), (7, 257, 8), (5, 512, 10),
                                   (3, 513, 1), (4, 1000, 16), (2, 1024, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_sizes(cuda, T, E, k, score, with_bias):
    x = logits(T, E, T + E, cuda)
    bias = None
    if with_bias:
        bias = torch.tensor(np.random.default_rng(E).standard_normal(E) * 0.1, dtype=torch.float32, device=cuda)
    check(x, k, bias, score=score, renormalize=k % 2 == 0, grad_seed=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_types_and_gradients(cuda, dtype, score, renormalize):
    check(logits(70, 48, 5, cuda, dtype), 4, score=score, renormalize=renormalize, scale=2.5, grad_seed=2)


@pytest.mark.parametrize("E,groups,top_groups", [(8, 8, 3), (64, 8, 4), (256, 8, 4), (60, 4, 1), (160, 8, 3),
                                                 (128, 64, 5), (1024, 64, 8), (6, 2, 2), (1000, 40, 7)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("score,with_bias", [("sigmoid", True), ("sigmoid", False), ("softmax", True),
                                             ("softmax", False)])
def test_groups(cuda, E, groups, top_groups, best, score, with_bias):
    bias = None
    if with_bias:
        bias = torch.tensor(np.random.default_rng(E).standard_normal(E) * 0.1, dtype=torch.float32, device=cuda)
    check(logits(21, E, E + groups, cuda), min(6, top_groups * (E // groups)), bias, score=score,
          groups=groups, top_groups=top_groups, group_best=best)


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_go_to_the_lowest_index(cuda, groups, with_bias):
    rng = np.random.default_rng(6)
    x = torch.tensor(rng.integers(-2, 3, (64, 96)), dtype=torch.bfloat16, device=cuda)
    x = torch.where(x == 0, torch.tensor(-0.0, dtype=x.dtype, device=cuda) * (x + 1), x)  # 0 and -0
    bias = torch.zeros(96, device=cuda) if with_bias else None
    for score in ("softmax", "sigmoid"):
        check(x, 8, bias, score=score, groups=groups, top_groups=max(1, groups // 2), group_best=2)


def test_scores_that_round_to_the_same_value(cuda):
    """Sigmoid scores near 1 tie in fp32 with a bias; without one the logits still tell them apart."""
    x = torch.linspace(18, 30, 32, device=cuda).flip(0).repeat(3, 1).contiguous()
    x[1] = x[1].flip(0)
    e, _ = check(x, 4, torch.zeros(32, device=cuda), score="sigmoid")
    assert e[1].tolist() == [0, 1, 2, 3]
    e, _ = check(x, 4, score="sigmoid")
    assert e[1].tolist() == [31, 30, 29, 28]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_masked_infinite_and_nan_logits(cuda, score, renormalize, with_bias):
    x = logits(10, 20, 7, cuda)
    x[0, 3:] = -torch.inf        # fewer experts left than are asked for
    x[1] = -torch.inf            # none left
    x[2, 4] = torch.nan
    x[3, 5] = torch.inf
    x[4] = torch.nan
    x[5, :] = torch.finfo(torch.float32).min
    x[6, ::2] = -200             # far below the others, and a sigmoid that underflows in fp32
    x[7] = -1000.0 - torch.arange(20, device=cuda)
    x[8, 0] = 3e38
    bias = torch.zeros(20, device=cuda) if with_bias else None
    if with_bias:
        bias[2], bias[7], bias[9] = -torch.inf, torch.inf, torch.nan
    check(x, 5, bias, score=score, renormalize=renormalize)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_masked_logits_have_gradients_that_are_numbers(cuda, score, renormalize):
    x = logits(4, 20, 8, cuda)
    x[0, 3:] = -torch.inf
    x[1] = -torch.inf
    x[2] = -1000.0 - torch.arange(20, device=cuda)
    x[3, 0] = 3e38
    x.requires_grad_()
    _, w = ops.route_experts(x, 5, score=score, renormalize=renormalize)
    g = torch.ones_like(w) + torch.arange(5, device=cuda)
    (dx,) = torch.autograd.grad(w, x, g)
    ids = O.choose(f64(x), 5, score)
    want = O.route_backward(f64(x), ids, f64(g), score, renormalize)
    assert dx.isfinite().all()
    np.testing.assert_allclose(f64(dx), want, rtol=1e-6, atol=16 * 15 * 2.0 ** -24)


@pytest.mark.parametrize("renormalize", [False, True])
def test_softmax_rows_without_weights_have_no_gradient(cuda, renormalize):
    """A NaN or +infinity anywhere in a softmax row makes its weights NaN, and their gradients: of all its
    logits, or of the chosen ones where the weights go by those alone."""
    x = logits(5, 20, 11, cuda)
    x[0, 4], x[1, 7], x[2, 3:] = torch.nan, torch.inf, torch.nan
    x.requires_grad_()
    e, w = ops.route_experts(x, 3, renormalize=renormalize)
    (dx,) = torch.autograd.grad(w, x, torch.ones_like(w))
    assert w[:3].isnan().all() and not w[3:].isnan().any() and not dx[3:].isnan().any()
    picked = dx[:3].gather(1, e[:3].long())
    assert picked.isnan().all()
    if renormalize:
        assert int(dx[:3].isnan().sum()) == 9 and int((dx[:3] == 0).sum()) == 51
    else:
        assert dx[:3].isnan().all()


def test_strides_leading_axes_and_no_tokens(cuda):
    big = logits(24, 50, 9, cuda)
    x = big[:, 5:37]
    e, w = ops.route_experts(x, 4)
    e2, w2 = ops.route_experts(x.reshape(2, 3, 4, 32).contiguous(), 4)
    e3, w3 = ops.route_experts(big.t()[5:37].t().contiguous().t().contiguous().t(), 4)
    assert e2.shape == (2, 3, 4, 4)
    for a, b in ((e, e2), (w, w2), (e, e3), (w, w3)):
        assert torch.equal(a.flatten(), b.flatten())
    wide = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(ops.route_experts(wide, 4)[1], wide, torch.arange(96., device=cuda).view(24, 4))
    dense = x.contiguous().requires_grad_()
    (dy,) = torch.autograd.grad(ops.route_experts(dense, 4)[1], dense, torch.arange(96., device=cuda).view(24, 4))
    assert torch.equal(dx, dy)
    e, w = ops.route_experts(torch.empty(0, 8, device=cuda), 2)
    assert e.shape == w.shape == (0, 2)
    none = torch.empty(0, 8, device=cuda, requires_grad=True)
    (d,) = torch.autograd.grad(ops.route_experts(none, 2)[1].sum(), none)
    assert d.shape == (0, 8)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_against_differences(cuda, score, renormalize):
    x = logits(6, 16, 10, cuda)
    x.requires_grad_()
    e, w = ops.route_experts(x, 3, score=score, renormalize=renormalize)
    g = torch.randn(w.shape, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    (dx,) = torch.autograd.grad(w, x, g)
    a = torch.randn(x.shape, device=cuda, generator=torch.Generator(cuda).manual_seed(2))
    step = 2.0 ** -6
    up, down = (ops.route_experts(x.detach() + s * a, 3, score=score, renormalize=renormalize)
                for s in (step, -step))
    same = ((up[0] == e) & (down[0] == e)).all(-1)  # a choice that changes has no derivative
    assert same.sum() >= 3
    slope = ((up[1] - down[1]) / (2 * step) * g).double().sum(-1)[same]
    want = (dx * a).double().sum(-1)[same]
    # third derivatives times step^2 / 6 (of functions bounded by 1, in directions of size 4), fp32 / step
    assert (slope - want).abs().max() < 64 * step ** 2 / 6 * 3


def test_refusals(cuda):
    x = torch.zeros(4, 8, device=cuda)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.route_experts(x.double(), 2)
    with pytest.raises(RuntimeError, match="bias must"):
        ops.route_experts(x, 2, bias=torch.zeros(7, device=cuda))
    with pytest.raises(RuntimeError, match="bias must"):
        ops.route_experts(x, 2, bias=torch.zeros(8, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="bias must"):
        ops.route_experts(x, 2, bias=torch.zeros(8))
    with pytest.raises(RuntimeError, match="top_k"):
        ops.route_experts(x, 9)
    with pytest.raises(RuntimeError, match="logits must be"):
        ops.route_experts(torch.zeros((), device=cuda), 1)
    x.requires_grad_()
    _, w = ops.route_experts(x, 2)
    (d,) = torch.autograd.grad(w.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        d.sum().backward()
