"""The weighted sum and its gradients at the sizes of training prompts, where a wave has a token, and of outputs
past the caches."""
import numpy as np
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu


def make(cuda, T, k, N, dtype, seed, E=7):
    gen = torch.Generator(cuda).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=cuda, generator=gen)
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device=cuda, generator=gen)
    g = ops.group_experts(ids, E)
    places = torch.where(rand(T, k) > 1.3, -1, g.places)  # some are taken away
    return (rand(T * k, N).to(dtype), rand(T, k), ops.ExpertGroups(g.offsets, g.entries, places),
            rand(T, N).to(dtype), rand(T, N).to(dtype))


def rows_of(y, places):
    """y's rows in 64 bits [T, k, N], 0 without a place."""
    held = places >= 0
    return y.detach().double()[places.clamp(min=0).long()] * held[..., None]


# 4096 tokens and more: each has a wave; the last workgroup is partly filled; top_k is no multiple of the rows that
# are taken together; rows start at any element
@pytest.mark.parametrize("T", [4095, 4096, 4097])
@pytest.mark.parametrize("k,N", [(1, 515), (3, 1000), (4, 77), (8, 1000), (10, 520), (3, 2041)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients(cuda, T, k, N, dtype):
    y, w, g, r, d = make(cuda, T, k, N, dtype, T + N + k)
    leaves = [t.requires_grad_() for t in (y, w, r)]
    out = ops.experts_combine(y, w, g, residual=r)
    dy, dw, dr = torch.autograd.grad(out, leaves, d)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    rows, d64, w64 = rows_of(y, g.places), d.double(), w.detach().double()
    parts = rows * w64[..., None]
    want, size = parts.sum(1) + r.detach().double(), parts.abs().sum(1) + r.detach().double().abs()
    # one rounding for each row's fused product and sum, one for the residual, one to y's type
    assert ((out.double() - want).abs() <= half * want.abs() + (k + 2) * 2.0 ** -24 * 1.01 * size + tiny).all()
    # a sum of N products: none of its partial sums is off by more than N + 8 half steps of their size
    want, size = (rows * d64[:, None]).sum(-1), (rows * d64[:, None]).abs().sum(-1)
    assert ((dw.double() - want).abs() <= (N + 8) * 2.0 ** -24 * 1.01 * size).all()
    want = torch.zeros(T * k, N, dtype=torch.float64, device=cuda)
    t, j = (g.places >= 0).nonzero(as_tuple=True)
    want[g.places[t, j].long()] = w64[t, j, None] * d64[t]
    assert ((dy.double() - want).abs() <= (half + 2.0 ** -24) * 1.01 * want.abs() + tiny).all()
    assert torch.equal(dr, d)


@pytest.mark.parametrize("T,k,N,dtype", [(9000, 8, 2041, torch.bfloat16), (8500, 8, 2044, torch.float16),
                                         (5000, 7, 2003, torch.float32), (30000, 3, 1500, torch.bfloat16)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_large_inputs(cuda, T, k, N, dtype, with_residual):
    """Rows of more than 256 MB are read past the caches; their ends and rows at any element too."""
    y, w, g, r, _ = make(cuda, T, k, N, dtype, N)
    assert y.numel() * y.element_size() >= 256 << 20
    out = ops.experts_combine(y, w, g, residual=r if with_residual else None)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for a in range(0, T, 3000):
        parts = rows_of(y, g.places[a:a + 3000]) * w[a:a + 3000, :, None].double()
        want, size = parts.sum(1), parts.abs().sum(1)
        if with_residual:
            want, size = want + r[a:a + 3000].double(), size + r[a:a + 3000].double().abs()
        off = (out[a:a + 3000].double() - want).abs()
        assert (off <= half * want.abs() + (k + 2) * 2.0 ** -24 * 1.01 * size + tiny).all()
