"""silu of the experts' product against the function in 64 bits; the other activations have the same bits as in the
product with one weight."""
import numpy as np
import pytest
import torch

import decoder_ops
import expert_ops as ops

pytestmark = pytest.mark.gpu


# few rows (aligned or not), tiles of 128 weight rows, tiles of 256
@pytest.mark.parametrize("T,N,K", [(8, 200, 64), (5, 33, 3), (600, 200, 64), (600, 130, 5), (9000, 4096, 16)])
def test_against_the_function_in_64_bits(cuda, T, N, K):
    # the first code and weight of a row are 1, the others 0: each value is a weight's scale, exactly
    v = torch.linspace(-80, 80, N, device=cuda) + 0.375
    v[:7] = torch.tensor([-1e-3, -1.0, -0.5, 0.25, -20.0, -60.0, 30.0], device=cuda)
    x = torch.zeros(T, K, dtype=torch.int8, device=cuda)
    w = torch.zeros(1, N, K, dtype=torch.int8, device=cuda)
    x[:, 0], w[:, :, 0] = 1, 1
    g = ops.group_experts(torch.zeros(T, 1, dtype=torch.int32, device=cuda), 1)
    y = ops.experts_linear_int8(x, torch.ones(T, device=cuda), w, v[None].contiguous(), g, activation="silu",
                                dtype=torch.float32)
    a = v.double().cpu().numpy()
    want = a / (1 + np.exp(-a))
    # exp(-|v|) within 3 half steps of fp32 (2^t within 1 ulp, what the rounding of t left is added back, rounded); its
    # product with v, its sum with 1, that one's reciprocal and the last product one each
    for row in (0, T // 2, T - 1):
        off = np.abs(y[row].double().cpu().numpy() - want) / np.abs(want)
        assert off.max() <= 7 * 2.0 ** -24 * 1.01, (off.max() * 2 ** 24, a[off.argmax()])
    assert torch.equal(y, y[:1].expand(T, -1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,N,K", [(8, 200, 64), (600, 130, 5), (9000, 4096, 16)])
@pytest.mark.parametrize("gated", [False, True])
def test_in_16_bits(cuda, T, N, K, dtype, gated):
    """Off by the rounding to the output's type and a small part of it."""
    v = torch.linspace(-30, 30, N, device=cuda) + 0.375
    x = torch.zeros(T, K, dtype=torch.int8, device=cuda)
    w = torch.zeros(1, N * (1 + gated), K, dtype=torch.int8, device=cuda)
    x[:, 0], w[:, :, 0] = 1, 1
    sw = torch.cat([v, torch.full_like(v, 0.75)]) if gated else v
    g = ops.group_experts(torch.zeros(T, 1, dtype=torch.int32, device=cuda), 1)
    y = ops.experts_linear_int8(x, torch.ones(T, device=cuda), w, sw[None].contiguous(), g, activation="silu",
                                gated=gated, dtype=dtype)
    a = v.double().cpu().numpy()
    want = a / (1 + np.exp(-a)) * (0.75 if gated else 1)
    # |v| + 4 half steps of fp32, the product's, and the output's
    bound = (torch.finfo(dtype).eps / 2 + (np.abs(a) + 5) * 2.0 ** -24) * 1.01 * np.abs(want)
    bound += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    off = np.abs(y[0].double().cpu().numpy() - want)
    assert (off <= bound).all(), (off / bound).max()
    assert torch.equal(y, y[:1].expand(T, -1))


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("T", [8, 600, 9000])
def test_one_expert_is_the_product_with_one_weight(cuda, act, T):
    gen = torch.Generator(cuda).manual_seed(T)
    rand = lambda *s: torch.randint(-127, 128, s, dtype=torch.int8, device=cuda, generator=gen)
    K, N = 96, 2048 if T > 1000 else 150
    x, w = rand(T, K), rand(1, 2 * N, K)
    sx = torch.rand(T, device=cuda, generator=gen) / 127
    sw = torch.rand(1, 2 * N, device=cuda, generator=gen) * 8 / 127
    b = torch.randn(1, 2 * N, device=cuda, generator=gen)
    g = ops.group_experts(torch.zeros(T, 1, dtype=torch.int32, device=cuda), 1)
    for bias in (None, b):
        one = lambda rows, act: decoder_ops.linear_int8(x, sx, w[0, rows], sw[0, rows],
                                                        None if bias is None else bias[0, rows], act,
                                                        dtype=torch.float32)
        kw = dict(activation=act, dtype=torch.float32)
        assert torch.equal(ops.experts_linear_int8(x, sx, w, sw, g, bias, **kw), one(slice(None), act))
        assert torch.equal(ops.experts_linear_int8(x, sx, w, sw, g, bias, gated=True, **kw),
                           one(slice(0, N), act) * one(slice(N, None), None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [8, 600])
def test_ends_of_the_range(cuda, T, dtype):
    big = torch.finfo(dtype).max
    v = torch.tensor([0.0, -0.0, 87.0, 200.0, big, torch.inf, -95.0, -1000.0, -big, torch.nan, -torch.inf], device=cuda)
    x = torch.ones(T, 1, dtype=torch.int8, device=cuda)
    g = ops.group_experts(torch.zeros(T, 1, dtype=torch.int32, device=cuda), 1)
    y = ops.experts_linear_int8(x, torch.ones(T, device=cuda), torch.ones(1, 11, 1, dtype=torch.int8, device=cuda),
                                v[None].contiguous(), g, activation="silu", dtype=dtype)
    assert torch.equal(y, y[:1].expand(T, -1)) or torch.equal(y.isnan(), y[:1].isnan().expand(T, -1))
    assert torch.equal(y[0, :6], v[:6].to(dtype)) and y[0, 9:].isnan().all()
    assert (y[0, 6:9].abs() < 1e-36).all()
