"""A feed-forward of experts in 8 bits on the GPU: routing, order, products and sums together, alone and in
a decoder layer, captured, on other streams; the training forms together."""
import math

import pytest
import torch

import decoder_ops as ops
import expert_ops
from quant_decoder import KVCache, QuantDecoderLayer, QuantExperts, Step

pytestmark = pytest.mark.gpu

WIDTH, HIDDEN, E, K = 128, 192, 12, 3


def floats(cuda, gated, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(cuda)
    return rand(E, WIDTH) * 3, rand(E, HIDDEN * (1 + gated), WIDTH), rand(E, WIDTH, HIDDEN)


def rows(n, cuda, seed=1):
    return torch.randn(n, WIDTH, generator=torch.Generator().manual_seed(seed)).to(cuda).bfloat16()


def in_64_bits(w_up, w_down, x, experts, weights, gated):
    """The chosen experts' sums on float weights."""
    x, out = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for j in range(experts.shape[1]):
        for e in range(len(w_up)):
            t = (experts[:, j] == e).nonzero()[:, 0]
            u = x[t] @ w_up[e].double().t()
            u = u[:, :HIDDEN] * torch.sigmoid(u[:, :HIDDEN]) * (u[:, HIDDEN:] if gated else 1)
            out[t] += weights[t, j, None].double() * (u @ w_down[e].double().t())
    return out


@pytest.mark.parametrize("tokens", [1, 16, 300])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("choice", [dict(), dict(score="sigmoid", with_bias=True, groups=4, top_groups=2,
                                                 group_best=2, scale=2.0)])
def test_against_float_experts(cuda, tokens, gated, choice):
    w = floats(cuda, gated)
    kw = dict(choice)
    bias = torch.linspace(-0.2, 0.2, E, device=cuda) if kw.pop("with_bias", False) else None
    m = QuantExperts.from_float(*w, top_k=K, gated=gated, bias=bias, **kw)
    x = rows(tokens, cuda)
    codes, scales = ops.quantize_rows(x)
    y = m(codes, scales)
    logits = ops.linear_int8(codes, scales, m.w_router, m.s_router, dtype=torch.float32)
    chosen, weights = expert_ops.route_experts(logits, K, bias=bias, **m.choice)
    want = in_64_bits(*w[1:], codes.double() * scales[:, None].double(), chosen, weights, gated)
    # Operands are rounded to 127 steps of a row whose largest value is some 3 standard deviations: 0.7 % of
    # noise each; the weights of both products, the gated product's two factors and the values between
    # them, and bf16 outputs (0.2 % twice): below 5 % of the sum's norm
    off = (y.double() - want).norm() / want.norm()
    assert off < 0.05, off
    assert torch.equal(m(codes, scales, residual=x * 0), y)
    r = rows(tokens, cuda, 2)
    both = m(codes, scales, residual=r)
    assert (both.double() - y.double() - r.double()).norm() < 2.0 ** -7 * (y.double().norm() + r.double().norm())


def test_tokens_do_not_go_by_each_other(cuda):
    """A token's result is the same alone, in a small and in a large batch: sums over K are exact, and the
    rest is made of the token's own values in a fixed order."""
    m = QuantExperts.from_float(*floats(cuda, True), top_k=K)
    x = rows(2000, cuda)
    codes, scales = ops.quantize_rows(x)
    all_ = m(codes, scales)
    for n in (1, 40, 700):
        assert torch.equal(m(codes[:n], scales[:n]), all_[:n])


@pytest.mark.parametrize("tokens", [4, 200])
def test_captured_and_replayed(cuda, tokens):
    m = QuantExperts.from_float(*floats(cuda, True), top_k=K)
    x = rows(tokens, cuda)
    run = lambda: m(*ops.quantize_rows(x), residual=x)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        y2 = run()
    for seed in (5, 6, 7):
        x.copy_(rows(tokens, cuda, seed))
        want = run()
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(y2, want)


def test_backward_captured_and_replayed(cuda):
    x = torch.randn(300, E, device=cuda, requires_grad=True)
    y = torch.randn(300 * K, 70, device=cuda, requires_grad=True)
    grad = torch.randn(300, 70, device=cuda)

    def run():
        experts, weights = expert_ops.route_experts(x, K, renormalize=False)
        out = expert_ops.experts_combine(y, weights, expert_ops.group_experts(experts, E))
        return torch.autograd.grad(out, (x, y), grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in (1, 2, 3):
        with torch.no_grad():
            x.copy_(torch.randn(300, E, generator=torch.Generator().manual_seed(seed)))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_another_stream(cuda):
    m = QuantExperts.from_float(*floats(cuda, False), top_k=K, gated=False)
    x = rows(500, cuda)
    codes, scales = ops.quantize_rows(x)
    want = m(codes, scales)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(m(codes, scales))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_router_and_sum_train_together(cuda):
    """Gradients of a float feed-forward of experts, routed and added up by the operators, against 64 bits."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, WIDTH, generator=g).to(cuda).requires_grad_()
    router = (torch.randn(E, WIDTH, generator=g) / math.sqrt(WIDTH)).to(cuda).requires_grad_()
    w = (torch.randn(E, WIDTH, WIDTH, generator=g) / math.sqrt(WIDTH)).to(cuda).requires_grad_()
    grad = torch.randn(40, WIDTH, generator=g).to(cuda)
    experts, weights = expert_ops.route_experts(x @ router.t(), K)
    groups = expert_ops.group_experts(experts, E)
    held = groups.entries.long() // K
    expert = torch.repeat_interleave(torch.arange(E, device=cuda), groups.offsets.diff().long())
    y = (x[held][:, None] @ w[expert].transpose(1, 2).contiguous())[:, 0]
    out = expert_ops.experts_combine(y, weights, groups, residual=x)
    got = torch.autograd.grad(out, (x, router, w), grad)

    x2, r2, w2 = (t.detach().double().requires_grad_() for t in (x, router, w))
    s = torch.softmax(torch.gather(x2 @ r2.t(), 1, experts.long()), -1)
    out2 = x2 + sum(s[:, j, None] * (x2[:, None] @ w2[experts[:, j].long()].transpose(1, 2).contiguous())[:, 0]
                    for j in range(K))
    want = torch.autograd.grad(out2, (x2, r2, w2), grad.double())
    assert (out.double() - out2).norm() < 1e-5 * out2.norm()
    for a, b in zip(got, want):
        # fp32 products over 128 terms: their sums' roundings are some 128 half steps at most
        assert (a.double() - b).norm() < 128 * 2.0 ** -24 * 4 * b.norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_in_a_decoder_layer(cuda, dtype):
    """Prompts and single tokens through a layer with experts."""
    g = torch.Generator().manual_seed(4)
    rand = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(cuda).to(dtype)
    ones = torch.ones(WIDTH, device=cuda).to(dtype)
    m = QuantExperts.from_float(*floats(cuda, True), top_k=K, dtype=dtype)
    layer = QuantDecoderLayer.from_float(ones, rand(256, WIDTH), rand(WIDTH, 128), ones, heads=2, kv_heads=1,
                                         experts=m, dtype=dtype)
    assert sorted(layer.state_dict()) == sorted(
        ["w_qkv", "s_qkv", "w_o", "s_o", "norm1", "norm2"]
        + [f"experts.{p}_{n}" for p in "ws" for n in ("router", "up", "down")])
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    x = torch.randn(20, WIDTH, generator=g).to(cuda).to(dtype)
    cache = KVCache.empty(2, 1, 64, 16, device=cuda)
    table = ints(0, 1)[None]
    whole = layer(x, cache, Step(table, ints(0), ints(0, 20), 20, 20))
    cache = KVCache.empty(2, 1, 64, 16, device=cuda)
    first = layer(x[:19], cache, Step(table, ints(0), ints(0, 19), 19, 20))
    last = layer(x[19:], cache, Step(table, ints(19), max_length=20))
    assert whole.isfinite().all() and whole.shape == x.shape and whole.dtype == dtype
    # the first 19 tokens see the same cache but for its page's scale, which the last one may raise
    got = torch.cat([first, last])
    assert (got.double() - whole.double()).norm() < 0.03 * whole.double().norm()
    assert layer(x[:0], cache, Step(table, ints(20), ints(0, 0), 0, 20)).shape == (0, WIDTH)


def test_refusals(cuda):
    w = floats(cuda, True)
    with pytest.raises(ValueError, match="w_up"):
        QuantExperts.from_float(*w, top_k=K, gated=False)
    with pytest.raises(ValueError, match="top_k"):
        QuantExperts.from_float(*w, top_k=E + 1)
    m = QuantExperts.from_float(*w, top_k=K)
    with pytest.raises(ValueError, match="width and dtype"):
        QuantDecoderLayer(64, 2, 1, 64, None, experts=m, device=cuda)
    with pytest.raises(ValueError, match="width and dtype"):
        QuantDecoderLayer(WIDTH, 2, 1, 64, None, experts=m, dtype=torch.float16, device=cuda)
    with pytest.raises(ValueError, match="either hidden or experts"):
        QuantDecoderLayer(WIDTH, 2, 1, 64, 64, experts=m, device=cuda)
