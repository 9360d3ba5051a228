"""The decoder operators under tracing, saved-tensor hooks, changed operands and second derivatives, through
the node in C++ and through the Python function."""
import pytest
import torch

import decoder_ops as ops

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["c++", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(ops, "_ext", False)
    else:
        assert ops._native(), "the module rxmet_torch is missing"
    return request.param


def make(cuda, rows=6, cols=200, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g).to(dtype).to(cuda).requires_grad_()
    r = torch.randn(rows, cols, generator=g).to(dtype).to(cuda).requires_grad_()
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype).to(cuda).requires_grad_()
    return x, w, r


# ---------------------------------------------------------------------------------
# Tracing
# ---------------------------------------------------------------------------------

@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("with_residual", [True, False])
def test_traced_training_form_runs_on_other_inputs(cuda, path, with_residual):
    x, w, r = (t.detach() for t in make(cuda))
    f = (lambda x, w, r: ops.rms_norm_quantize_dequantize(x, w, r)) if with_residual else \
        (lambda x, w, r: ops.rms_norm_quantize_dequantize(x, w))
    traced = torch.jit.trace(f, (x, w, r), check_trace=False)
    for seed in (1, 2):
        args = [t.detach() for t in make(cuda, seed=seed)]
        for a, b in zip(traced(*args), f(*args)):
            assert torch.equal(a, b)


@pytest.mark.filterwarnings("ignore")
def test_serving_calls_refuse_a_trace(cuda, path):
    x, w, _ = (t.detach() for t in make(cuda, cols=64))
    codes, scales = ops.quantize_rows(x)
    cache = ops.KVCache.empty(1, 1, 64, 16, device=cuda)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    table, zero = ints(0)[None], ints(0)
    q = x[:1, None].half()
    ops.kv_cache_append(cache, q, q, table, zero)
    for f in (lambda x: ops.rms_norm_quantize(x, w)[1], lambda x: ops.quantize_rows(x)[1],
              lambda x: ops.linear_int8(codes, scales, codes, scales, dtype=torch.float32) + x[0, 0],
              lambda x: ops.kv_cache_append(cache, x[:1, None], x[:1, None], table, zero) or x,
              lambda x: ops.kv_cache_read(cache, table, zero, ints(0, 1), 1)[0] + x[0, 0],
              lambda x: ops.kv_cache_attention(x[:1, None].half(), cache, table, zero + 1)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
        f(x)  # outside a trace as ever


def test_transforms_are_refused(cuda, path):
    x, w, r = make(cuda)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: ops.rms_norm_quantize_dequantize(x, w.detach())[0])(x.detach()[None])
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        ops.rms_norm_quantize_dequantize(fwAD.make_dual(x.detach().requires_grad_(), torch.ones_like(x)), w)


# ---------------------------------------------------------------------------------
# Saved tensors
# ---------------------------------------------------------------------------------

def gradients(y, h, inputs):
    return torch.autograd.grad([y, h], inputs, [torch.ones_like(y) * 0.5, torch.ones_like(h)])


def test_hooks_that_keep_the_values(cuda, path):
    """Saved tensors on the host, or strided, in the meantime: the same gradients."""
    x, w, r = make(cuda)
    inputs = (x, w, r)
    ref = gradients(*ops.rms_norm_quantize_dequantize(*inputs), inputs)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: (seen.append(tuple(t.shape)), t.cpu())[1], lambda t: t.to(cuda)):
        out = ops.rms_norm_quantize_dequantize(*inputs)
    assert seen == [(6, 200), (200,), (6,)]
    assert all(torch.equal(a, b) for a, b in zip(gradients(*out, inputs), ref))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0]):
        out = ops.rms_norm_quantize_dequantize(*inputs)
    assert all(torch.equal(a, b) for a, b in zip(gradients(*out, inputs), ref))


@pytest.mark.parametrize("which", [0, 1, 2])  # h, weight, rstd
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.double(), lambda t: t.half(),
                                    lambda t: t[:-1], lambda t: t[..., None], lambda t: t.new_zeros(())],
                         ids=["host", "double", "half", "short", "axis", "scalar"])
def test_hooks_that_give_back_something_else(cuda, path, which, change):
    """Another device, type or shape is refused before anything is read."""
    inputs = make(cuda)
    count = iter(range(100))
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: (next(count), t), lambda p: change(p[1]) if p[0] == which else p[1]):
        out = ops.rms_norm_quantize_dequantize(*inputs)
    with pytest.raises(RuntimeError, match="saved"):
        gradients(*out, inputs)


def test_changed_operands_and_second_backward_are_refused(cuda, path):
    x, w, r = make(cuda)
    out = ops.rms_norm_quantize_dequantize(x, w, r)
    gradients(*out, (x, w, r))
    with pytest.raises(RuntimeError, match="second time"):
        gradients(*out, (x, w, r))
    out = ops.rms_norm_quantize_dequantize(x, w)
    with torch.no_grad():
        x.mul_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        gradients(*out, (x, w))


# ---------------------------------------------------------------------------------
# Second derivatives
# ---------------------------------------------------------------------------------

@pytest.mark.parametrize("with_residual", [True, False])
def test_second_derivatives_are_refused(cuda, path, with_residual):
    """A penalty on the gradient raises, alone and beside a term that has a gradient, whatever input it is
    taken in; the gradients themselves are those of an ordinary backward."""
    x, w, r = make(cuda)
    inputs = (x, w, r) if with_residual else (x, w)
    ref = torch.autograd.grad(ops.rms_norm_quantize_dequantize(*inputs)[0].square().sum(), inputs)
    for k in range(len(inputs)):
        y, _ = ops.rms_norm_quantize_dequantize(*inputs)
        grads = torch.autograd.grad(y.square().sum(), inputs, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, ref))
        with pytest.raises(RuntimeError, match="twice"):
            (y.sum() + grads[k].square().sum()).backward()
    y, _ = ops.rms_norm_quantize_dequantize(*inputs)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)  # an incoming gradient without one of its own
    with pytest.raises(RuntimeError, match="twice"):
        (y.sum() + g.square().sum()).backward()


def test_second_derivative_of_a_frozen_weight(cuda, path):
    x, w, _ = make(cuda)
    w = w.detach()
    y, _ = ops.rms_norm_quantize_dequantize(x, w)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


# ---------------------------------------------------------------------------------
# Serving
# ---------------------------------------------------------------------------------

def test_serving_outputs_carry_no_gradient(cuda, path):
    """h is detached with a residual and without; it is x itself where that carries none."""
    x, w, r = make(cuda)
    for res in (None, r):
        codes, scales, h = ops.rms_norm_quantize(x, w, res)
        assert not (codes.requires_grad or scales.requires_grad or h.requires_grad)
    assert torch.equal(ops.rms_norm_quantize(x, w)[2], x.detach())
    assert ops.rms_norm_quantize(x.detach(), w)[2].data_ptr() == x.data_ptr()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_programs(cuda, backend):
    """Operators between the graphs of a compiled program give what they give without it."""
    assert ops._native(), "the module rxmet_torch is missing"
    x, w, _ = make(cuda, cols=64)
    codes, scales = ops.quantize_rows(x.detach())

    def train(x, w):
        y, h = ops.rms_norm_quantize_dequantize(x * 2, w)
        return (y * h).sum()

    def serve(x):
        c, s, h = ops.rms_norm_quantize(x * 2, w)
        return ops.linear_int8(c, s, codes, scales) * 2 + ops.quantize_rows(h)[1][0]

    torch._dynamo.reset()
    got, want = torch.compile(train, backend=backend)(x, w), train(x, w)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (x, w)), torch.autograd.grad(want, (x, w))):
        assert torch.equal(a, b)
    assert torch.equal(torch.compile(serve, backend=backend)(x.detach()), serve(x.detach()))
    torch._dynamo.reset()
