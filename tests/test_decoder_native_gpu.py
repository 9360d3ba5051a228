"""The decoder operators' calls in C++ against the same calls through ctypes: the same kernels on the
same operands, so every output is equal bit for bit; and what the C++ side leaves to the other."""
import pytest
import torch

import decoder_ops as ops

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
    return a


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_residual", [True, False])
def test_rows(cuda, monkeypatch, dtype, with_residual):
    x = torch.randn(3, 5, 130, device=cuda).to(dtype)
    r = torch.randn_like(x) if with_residual else None
    for w in (torch.rand(130, device=cuda).to(dtype), torch.rand(130, device=cuda)):
        both(monkeypatch, lambda: ops.rms_norm_quantize(x, w, r))
        both(monkeypatch, lambda: ops.quantize_rows(x))

        def train():
            leaves = [t.detach().clone().requires_grad_() for t in (x, w) + ((r,) if with_residual else ())]
            y, h = ops.rms_norm_quantize_dequantize(*leaves)
            return [y, h] + list(torch.autograd.grad([y, h], leaves, [torch.ones_like(y), y.detach()]))

        both(monkeypatch, train)


@pytest.mark.parametrize("M", [3, 40, 200])
@pytest.mark.parametrize("K", [96, 101])
def test_linear(cuda, monkeypatch, M, K):
    x = torch.randint(-127, 128, (M, K), dtype=torch.int8, device=cuda)
    w = torch.randint(-127, 128, (70, K), dtype=torch.int8, device=cuda)
    sx, sw = torch.rand(M, device=cuda), torch.rand(70, device=cuda)
    b, r = torch.randn(70, device=cuda), torch.randn(M, 70, device=cuda)
    both(monkeypatch, lambda: ops.linear_int8(x, sx, w, sw, dtype=torch.float32))
    both(monkeypatch, lambda: ops.linear_int8(x, sx, w, sw, b, "gelu", r, torch.float32))


def test_cache(cuda, monkeypatch):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    x = torch.randn(50, 2, 2, 64, device=cuda).bfloat16()
    table, cu = ints(0, 1, 2, 3).view(2, 2), ints(0, 30, 50)

    def run():
        cache = ops.KVCache(*[t.zero_() for t in ops.KVCache.empty(4, 2, 64, 32, device=cuda)])
        ops.kv_cache_append(cache, x[:, 0], x[:, 1], table, ints(0, 0), cu, 30)
        ops.kv_cache_append(cache, x[:2, 0], x[:2, 1], table, ints(30, 20))
        q = x[:, 0].repeat(1, 2, 1)
        return [*cache, *ops.kv_cache_read(cache, table, ints(0, 0), cu, 50),
                ops.kv_cache_attention(q, cache, table, ints(31, 21), cu, 30, 31, window=9),
                ops.kv_cache_attention(q[:2], cache, table, ints(31, 21), scale=0.3)]

    both(monkeypatch, run)


def test_what_needs_a_copy_or_has_no_rows(cuda, monkeypatch):
    wide = torch.randn(40, 90, device=cuda)
    w = torch.rand(180, device=cuda)[::2]
    both(monkeypatch, lambda: ops.rms_norm_quantize(wide, w))
    both(monkeypatch, lambda: ops.quantize_rows(wide.t()))
    both(monkeypatch, lambda: ops.quantize_rows(wide[:0]))
    both(monkeypatch, lambda: ops.quantize_rows(wide[::2, 3:40]))
