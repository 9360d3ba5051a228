"""The expert operators where offsets pass 32 bits: weights and rows of more than 2^31 elements."""
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 600])
def test_weights_beyond_32_bits(cuda, T):
    E, N, K = 40, 8192, 8192  # 2.7e9 bytes
    w = torch.zeros(E, N, K, dtype=torch.int8, device=cuda)
    w[-1, :, :] = 1
    w[-1, -1, :] = 2
    ids = torch.full((T, 1), E - 1, dtype=torch.int32, device=cuda)
    g = ops.group_experts(ids, E)
    x = torch.ones(T, K, dtype=torch.int8, device=cuda)
    y = ops.experts_linear_int8(x, torch.ones(T, device=cuda), w, torch.ones(E, N, device=cuda), g,
                                dtype=torch.float32)
    assert (y[:, :-1] == K).all() and (y[:, -1] == 2 * K).all()


def test_rows_beyond_32_bits(cuda):
    T, E, N, K = 300000, 4, 8192, 64  # 2.5e9 elements of y
    ids = (torch.arange(T, device=cuda, dtype=torch.int32) % E)[:, None].contiguous()
    g = ops.group_experts(ids, E)
    x = torch.ones(T, K, dtype=torch.int8, device=cuda)
    w = torch.ones(E, N, K, dtype=torch.int8, device=cuda) * torch.arange(1, E + 1, device=cuda, dtype=torch.int8)[:, None, None]
    y = ops.experts_linear_int8(x, torch.ones(T, device=cuda), w, torch.ones(E, N, device=cuda), g)
    # 64, 128, 192 and 256 are whole in bf16
    for e in range(E):
        a, b = int(g.offsets[e]), int(g.offsets[e + 1])
        for r in (a, (a + b) // 2, b - 1):
            assert (y[r] == K * (e + 1)).all()
    half = torch.full((T, 1), 0.5, device=cuda)
    out = ops.experts_combine(y, half, g)
    for t in (0, 1, T // 2 + 1, T - 2, T - 1):
        assert (out[t] == K * (t % E + 1) / 2).all()
    del out
    half.requires_grad_()
    y.requires_grad_()
    grad = torch.ones(1, 1, dtype=torch.bfloat16, device=cuda).expand(T, N)
    dy, dw = torch.autograd.grad(ops.experts_combine(y, half, g), (y, half), grad)
    assert (dy[0] == 0.5).all() and (dy[-1] == 0.5).all() and (dy[T // 2] == 0.5).all()
    want = K * N * (ids[:, 0] + 1).float()  # sums of equal whole numbers below 2^24
    assert torch.equal(dw[:, 0], want)
