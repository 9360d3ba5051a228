"""The router of a feed-forward of experts in 8 bits: its choice differs from a float router's on the same codes
only among experts whose logits lie within the weights' rounding of each other."""
import math

import pytest
import torch

import decoder_ops as ops
import expert_ops
from quant_decoder import QuantExperts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,E,k", [(128, 12, 3), (2048, 64, 8)])
def test_choices_differ_within_the_rounding(cuda, width, E, k):
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(cuda)
    router = rand(E, width)
    m = QuantExperts.from_float(router, rand(E, 32, width), rand(E, width, 16), top_k=k)
    codes, scales = ops.quantize_rows(torch.randn(1500, width, generator=g).to(cuda).bfloat16())
    logits = ops.linear_int8(codes, scales, m.w_router, m.s_router, dtype=torch.float32)
    experts, _ = expert_ops.route_experts(logits, k, **m.choice)
    x = codes.double() * scales[:, None].double()
    exact = x @ router.double().t().contiguous()
    # a weight is off by half a step of its row's grid, the scale by a rounding of fp32 in 127 steps at most; the
    # logits' own roundings are three of fp32
    size = x.abs().sum(-1, keepdim=True) * m.s_router.double()
    off = size * (0.5 + 127 * 2.0 ** -22) + 4 * 2.0 ** -24 * (exact.abs() + size)
    assert ((logits.double() - exact).abs() <= off).all()
    chosen = torch.zeros(1500, E, dtype=torch.bool, device=cuda).scatter_(1, experts.long(), True)
    least = torch.where(chosen, exact + off, torch.inf).amin(1)          # the least that is chosen, at its highest
    most = torch.where(chosen, -torch.inf, exact - off).amax(1)          # the largest that is not, at its lowest
    assert (least >= most).all()
    y = m(codes, scales)
    groups = expert_ops.group_experts(experts, E)  # and this is the choice that the module makes
    u = expert_ops.experts_linear_int8(codes, scales, m.w_up, m.s_up, groups, activation="silu", gated=True)
    u, s = ops.quantize_rows(u)
    out = expert_ops.experts_linear_int8(u, s, m.w_down, m.s_down, groups, grouped=True)
    assert torch.equal(y, expert_ops.experts_combine(out, expert_ops.route_experts(logits, k)[1], groups))
