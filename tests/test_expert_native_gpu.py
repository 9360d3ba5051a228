"""The expert operators' calls in C++ against the same calls through ctypes: the same kernels on the same
operands, so every output is equal bit for bit; and what the C++ side leaves to the other."""
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu


def both(monkeypatch, call):
    """call() with the C++ module and without it."""
    assert ops._native(), "the module rxmet_torch is missing"
    a = call()
    monkeypatch.setattr(ops, "_ext", False)
    b = call()
    monkeypatch.undo()
    flat = lambda v: v if isinstance(v, (list, tuple)) else [v]
    assert len(flat(a)) == len(flat(b))
    for x, y in zip(flat(a), flat(b)):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)
        assert x.requires_grad == y.requires_grad
    return a


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(cuda, monkeypatch, dtype, score):
    x = torch.randn(4, 10, 24, device=cuda).to(dtype)
    bias = torch.randn(24, device=cuda)
    for kw in (dict(), dict(bias=bias, renormalize=False, scale=0.5),
               dict(groups=4, top_groups=2, group_best=2, bias=bias.requires_grad_())):
        both(monkeypatch, lambda: ops.route_experts(x, 3, score=score, **kw))

        def train():
            v = x.detach().clone().requires_grad_()
            e, w = ops.route_experts(v, 3, score=score, **kw)
            assert not e.requires_grad
            return [e, w, *torch.autograd.grad(w, v, w.detach() + 1)]

        both(monkeypatch, train)
        with torch.no_grad():
            both(monkeypatch, lambda: ops.route_experts(x.clone().requires_grad_(), 3, score=score, **kw))


def sample(cuda, T=50, k=3, E=6):
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device=cuda)
    return ids, ops.group_experts(ids, E)


def test_groups(cuda, monkeypatch):
    ids, _ = sample(cuda, 3000)
    both(monkeypatch, lambda: ops.group_experts(ids, 6))
    both(monkeypatch, lambda: ops.group_experts(ids[::2, 1:], 6))
    both(monkeypatch, lambda: ops.group_experts(ids[:0], 6))


@pytest.mark.parametrize("gated,grouped", [(False, False), (True, False), (False, True)])
def test_linear(cuda, monkeypatch, gated, grouped):
    _, g = sample(cuda)
    held, rows = int(g.offsets[-1]), 150 if grouped else 50
    x = torch.randint(-127, 128, (rows, 96), dtype=torch.int8, device=cuda)
    w = torch.randint(-127, 128, (6, 40, 96), dtype=torch.int8, device=cuda)
    sx, sw, b = torch.rand(rows, device=cuda), torch.rand(6, 40, device=cuda), torch.randn(6, 40, device=cuda)
    run = lambda **kw: both(monkeypatch, lambda: ops.experts_linear_int8(
        **{**dict(codes=x, scales=sx, weight=w, weight_scales=sw, groups=g, gated=gated, grouped=grouped,
                  dtype=torch.float32), **kw})[:held])
    run()
    run(bias=b, activation="gelu")
    run(weight=w.transpose(1, 2).contiguous().transpose(1, 2), weight_scales=sw.t().contiguous().t())
    run(codes=x[:, 1:60], weight=w[:, :, 1:60])
    run(groups=g._replace(places=g.places.t().contiguous().t()))


def test_combine(cuda, monkeypatch):
    _, g = sample(cuda)
    y, w, r = torch.randn(150, 33, device=cuda), torch.rand(50, 3, device=cuda), torch.randn(50, 33, device=cuda)
    both(monkeypatch, lambda: ops.experts_combine(y, w, g))
    both(monkeypatch, lambda: ops.experts_combine(y.repeat(1, 2)[:, 3:36], w, g, residual=r))
    both(monkeypatch, lambda: ops.experts_combine(y.t().contiguous().t(), w.t().contiguous().t(), g, residual=r))

    def train(need):
        leaves = [t.detach().clone().requires_grad_(n) for t, n in zip((y, w, r), need)]
        out = ops.experts_combine(leaves[0], leaves[1], g, residual=leaves[2])
        return [out, *torch.autograd.grad(out, [t for t in leaves if t.requires_grad], r + 1)]

    for need in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        both(monkeypatch, lambda: train(need))


@pytest.mark.parametrize("native", [True, False])
def test_a_gradient_that_is_not_dense(cuda, monkeypatch, native):
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    _, g = sample(cuda)
    y = torch.randn(150, 32, device=cuda, requires_grad=True)
    w = torch.rand(50, 3, device=cuda, requires_grad=True)
    grad = torch.randn(32, 50, device=cuda).t()
    got = torch.autograd.grad(ops.experts_combine(y, w, g), (y, w), grad)
    want = torch.autograd.grad(ops.experts_combine(y, w, g), (y, w), grad.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(ops.experts_combine(y, w, g).sum(), (y, w))  # broadcast from one element
    want = torch.autograd.grad(ops.experts_combine(y, w, g), (y, w), torch.ones(50, 32, device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(50, 8, device=cuda, requires_grad=True)
    (a,) = torch.autograd.grad(ops.route_experts(x, 3)[1], x, torch.ones(3, 50, device=cuda).t() * 2)
    (b,) = torch.autograd.grad(ops.route_experts(x, 3)[1], x, torch.full((50, 3), 2.0, device=cuda))
    assert torch.equal(a, b)


@pytest.mark.parametrize("native", [True, False])
def test_unpack_hooks_traces_and_changed_inputs(cuda, monkeypatch, native):
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    _, g = sample(cuda)
    x = torch.randn(50, 8, device=cuda, requires_grad=True)
    y = torch.randn(150, 32, device=cuda, requires_grad=True)
    for change in (lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            w = ops.route_experts(x, 3)[1]
            out = ops.experts_combine(y, torch.rand(50, 3, device=cuda), g)
        for o, leaf in ((w, x), (out, y)):
            with pytest.raises(RuntimeError):
                torch.autograd.grad(o.sum(), leaf)
    w = ops.route_experts(x, 3)[1]
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()
    for f, args in ((lambda v: ops.route_experts(v, 2)[1], x.detach()),
                    (lambda v: ops.experts_combine(v, torch.ones(50, 3, device=cuda), g), y.detach())):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, args)


def test_saved_tensors_may_be_packed_elsewhere(cuda):
    _, g = sample(cuda)
    x = torch.randn(50, 8, device=cuda, requires_grad=True)
    y = torch.randn(150, 32, device=cuda, requires_grad=True)

    def run():
        out = ops.experts_combine(y, ops.route_experts(x, 3)[1], g)
        return out, torch.autograd.grad(out.sum(), (x, y))

    want = run()[1]
    with torch.autograd.graph.save_on_cpu():
        got = run()[1]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_programs(cuda, backend):
    """Operators between the graphs of a compiled program give what they give without it."""
    ids, g = sample(cuda)
    x = torch.randn(50, 8, device=cuda, requires_grad=True)
    y = torch.randn(150, 32, device=cuda, requires_grad=True)

    def train(x, y):
        e, w = ops.route_experts(x * 2, 3, renormalize=False)
        return (ops.experts_combine(y * 2, w, ops.group_experts(e, 8)) ** 2).sum()

    torch._dynamo.reset()
    got, want = torch.compile(train, backend=backend)(x, y), train(x, y)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (x, y)), torch.autograd.grad(want, (x, y))):
        assert torch.equal(a, b)
    torch._dynamo.reset()


def test_transforms_are_refused(cuda):
    _, g = sample(cuda)
    y, w = torch.randn(150, 32, device=cuda), torch.rand(50, 3, device=cuda)
    x = torch.randn(50, 8, device=cuda)
    for f, v in ((lambda v: ops.route_experts(v, 3)[1].sum(), x),
                 (lambda v: ops.experts_combine(v, w, g).sum(), y),
                 (lambda v: ops.experts_combine(y, w * v.sum(), g).sum(), x)):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(v)
