"""Gradient of a softmax router's weights as they are, held to the roundings of its outputs."""
import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k", [(40, 60, 4), (33, 200, 8), (9, 1000, 6), (1300, 64, 2), (1027, 128, 4), (1025, 500, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_rounded_once(cuda, T, E, k, dtype, spread):
    """With a large spread one expert has nearly all of the weight, and what is left of its gradient is the difference
    of numbers that are nearly the same."""
    gen = torch.Generator(cuda).manual_seed(T + E)
    x = (torch.randn(T, E, device=cuda, generator=gen) * spread).to(dtype).requires_grad_()
    ids, w = ops.route_experts(x, k, renormalize=False, scale=1.5)
    g = torch.randn(T, k, device=cuda, generator=gen)
    (dx,) = torch.autograd.grad(w, x, g)
    f64 = lambda t: t.detach().double().cpu().numpy()
    want = O.route_backward(f64(x), ids.cpu().numpy(), f64(g), "softmax", False, 1.5)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    # rounded to fp32 and to x's type; exp, sums and differences in 64 bits are off by 2^-44 of what they add up
    # (E + k terms, some 2^-52 each), here as in the oracle
    size = 1.5 * np.abs(f64(g)).sum(-1, keepdims=True) * O.scores(f64(x), "softmax")
    bound = (half + (2.0 ** -24 if dtype != torch.float32 else 0)) * 1.01 * np.abs(want) + 2.0 ** -42 * size + tiny
    off = np.abs(f64(dx) - want)
    assert (off <= bound).all(), (off / bound).max()
