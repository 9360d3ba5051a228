"""Routing of more than 1024 tokens, where several tokens share a wave, against the definition in 64 bits and
against the same tokens in small batches."""
import numpy as np
import pytest
import torch

import expert_ops as ops
from test_expert_route_gpu import TYPES, check, logits

pytestmark = pytest.mark.gpu

# both sides of each number of lanes and experts of a lane; token counts that leave a wave partly filled
EXPERTS = [1, 7, 64, 65, 128, 129, 256, 257, 512, 513, 1024]


def some_bias(E, cuda):
    return torch.tensor(np.random.default_rng(E).standard_normal(E) * 0.1, dtype=torch.float32, device=cuda)


@pytest.mark.parametrize("T", [1025, 1027])
@pytest.mark.parametrize("E", EXPERTS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sizes(cuda, T, E, score):
    for with_bias, renormalize in ((False, False), (True, True)):
        check(logits(T, E, T + E, cuda), min(E, 5), some_bias(E, cuda) if with_bias else None, score=score,
              renormalize=renormalize, scale=1.5, grad_seed=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [48, 100, 250, 400])
@pytest.mark.parametrize("renormalize", [False, True])
def test_types(cuda, dtype, E, renormalize):
    for score in ("softmax", "sigmoid"):
        check(logits(1026, E, 5, cuda, dtype), 8, score=score, renormalize=renormalize, grad_seed=2)


@pytest.mark.parametrize("E,groups,top_groups", [(8, 8, 3), (60, 4, 1), (64, 64, 9), (128, 2, 1), (160, 8, 3),
                                                 (256, 8, 4), (510, 3, 2), (512, 64, 8), (1024, 2, 1)])
@pytest.mark.parametrize("best", [1, 2])
def test_groups(cuda, E, groups, top_groups, best):
    for score, with_bias in (("sigmoid", True), ("softmax", True), ("softmax", False)):
        check(logits(1027, E, E + groups, cuda), min(6, top_groups * (E // groups)),
              some_bias(E, cuda) if with_bias else None, score=score, groups=groups, top_groups=top_groups, group_best=best)


@pytest.mark.parametrize("E", [60, 128, 250, 512])
@pytest.mark.parametrize("groups", [1, 2])
def test_ties(cuda, E, groups):
    x = torch.tensor(np.random.default_rng(6).integers(-2, 3, (1025, E)), dtype=torch.bfloat16, device=cuda)
    x = torch.where(x == 0, torch.tensor(-0.0, dtype=x.dtype, device=cuda) * (x + 1), x)  # 0 and -0
    for bias in (None, torch.zeros(E, device=cuda)):
        check(x, 8, bias, score="sigmoid", groups=groups, group_best=2)
        check(x, 8, bias, groups=groups, top_groups=1)


def spoiled(E, cuda):
    """Rows with NaN, infinities and nothing left between ordinary ones of the same wave."""
    x = logits(1027, E, E, cuda)
    n = torch.arange(1027, device=cuda)
    x[n % 7 == 1, E - 1] = torch.nan
    x[n % 7 == 2, 0] = torch.inf
    x[n % 7 == 3] = -torch.inf
    x[n % 7 == 4, 3:] = -torch.inf
    x[-1] = torch.nan
    return x


@pytest.mark.parametrize("E", [20, 128, 256, 500, 1000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_rows_do_not_spoil_their_neighbours(cuda, E, score, renormalize):
    x = spoiled(E, cuda)
    for bias in (None, some_bias(E, cuda)):
        check(x, 5, bias, score=score, renormalize=renormalize)
    x.requires_grad_()
    e, w = ops.route_experts(x, 5, score=score, renormalize=renormalize)
    g = torch.randn(w.shape, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    (dx,) = torch.autograd.grad(w, x, g)
    good = (x.isfinite() | (x == -torch.inf)).all(-1)
    assert dx[good].isfinite().all()
    # the same rows in batches that give each a wave of its own
    for i in range(0, 1027, 300):
        part = x.detach()[i:i + 300].requires_grad_()
        e2, w2 = ops.route_experts(part, 5, score=score, renormalize=renormalize)
        (d2,) = torch.autograd.grad(w2, part, g[i:i + 300])
        assert torch.equal(e2, e[i:i + 300])
        # sums in another order in 64 bits, then rounded to fp32: at most the next value
        for a, b in ((w[i:i + 300], w2), (dx[i:i + 300], d2)):
            torch.testing.assert_close(a, b, rtol=2.0 ** -22, atol=2.0 ** -22, equal_nan=True)


@pytest.mark.parametrize("E", [50, 120, 256, 500])
def test_rows_that_are_not_side_by_side(cuda, E):
    big = logits(1030, E + 30, 9, cuda)
    x = big[:, 11:11 + E]
    want = ops.route_experts(x.contiguous(), 4)
    assert all(torch.equal(a, b) for a, b in zip(ops.route_experts(x, 4), want))
    leaf, dense = x.detach().requires_grad_(), x.contiguous().requires_grad_()
    g = torch.arange(1030 * 4., device=cuda).view(1030, 4)
    (a,) = torch.autograd.grad(ops.route_experts(leaf, 4)[1], leaf, g)
    (b,) = torch.autograd.grad(ops.route_experts(dense, 4)[1], dense, g)
    assert torch.equal(a, b)
