"""The 8-bit decoder operators without a GPU: their oracle against itself, and what the library
refuses before any device call."""
import ctypes

import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O
import rxmet_lib


def test_oracle_gradient_is_the_smooth_norms_derivative():
    rng = np.random.default_rng(0)
    h, w, dy = rng.standard_normal((3, 17)), rng.standard_normal(17), rng.standard_normal((3, 17))
    dx, dw = O.rms_backward(h, w, 1e-3, dy, None)
    for k in range(5):
        a, b, t = rng.standard_normal(h.shape), rng.standard_normal(w.shape), 1e-5
        f = lambda s: (O.rms_smooth(h + s * a, w + s * b, 1e-3) * dy).sum()
        assert abs((f(t) - f(-t)) / (2 * t) - (dx * a).sum() - (dw * b).sum()) < 1e-7


def test_oracle_sees_a_planted_mistake():
    """The comparison that the GPU tests make fails where the oracle's own sums leave a term out."""
    rng = np.random.default_rng(1)
    h, w, dy = rng.standard_normal((3, 40)), rng.standard_normal(40), rng.standard_normal((3, 40))
    dx, _ = O.rms_backward(h, w, 1e-6, dy, None)
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6)
    without = rstd * dy * w  # the mean's part is missing
    assert np.abs(dx - without).max() > 1e-2


def test_oracle_codes_do_not_go_by_the_norm():
    rng = np.random.default_rng(2)
    h, w = rng.standard_normal((4, 33)), rng.standard_normal(33)
    q, scale, rstd = O.rms_quantize(h, w, 1e-6)
    assert np.allclose(q * scale[:, None], h * rstd[:, None] * w, rtol=1e-14)
    assert np.allclose(np.abs(q).max(-1), 127)


def test_oracle_attention_on_one_token():
    v = np.arange(4.0)[None]
    out, _ = O.attention(np.ones((1, 2, 4)), np.ones((1, 4)), np.ones(1), v, np.full(1, 0.5), 1, 1.0,
                         True, 0)
    assert np.array_equal(out, np.broadcast_to(0.5 * v, (1, 2, 4)))
    out, _ = O.attention(np.ones((2, 1, 4)), np.ones((1, 4)), np.ones(1), v, np.ones(1), 1, 1.0, True, 0)
    assert (out[0] == 0).all() and np.array_equal(out[1, 0], v[0])


def test_operators_refuse_host_tensors():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for f in (lambda: ops.rms_norm_quantize(x, w), lambda: ops.quantize_rows(x),
              lambda: ops.rms_norm_quantize_dequantize(x, w),
              lambda: ops.linear_int8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f()
    cache = ops.KVCache.empty(2, 1, 64, 16, device="cpu")
    with pytest.raises(RuntimeError, match="on the GPU"):
        ops.kv_cache_attention(x, cache, torch.zeros(1, 1, dtype=torch.int32), x)


def test_library_refuses_before_any_device_call():
    lib = rxmet_lib.load()
    buf = (ctypes.c_float * 16)()
    p = ctypes.addressof(buf) // 16 * 16

    def says(rc, text):
        assert rc == -22 and text in lib.rxmet_last_error().decode(), lib.rxmet_last_error()

    fwd = lambda rows, cols, dtype: lib.rxmet_rms_quantize_forward(
        p, cols, None, 0, p, 0, None, p, None, p, None, rows, cols, dtype, 1e-6, None)
    says(fwd(1, 0, 0), "cols between 1 and 65536")
    says(fwd(1, 65537, 0), "cols between 1 and 65536")
    says(fwd(1, 8, 3), "fp32, fp16 or bf16")
    says(lib.rxmet_rms_quantize_forward(p, 8, p, 8, p, 0, None, p, None, p, None, 1, 8, 0, 1e-6,
                                        None), "residual needs")
    lin = lambda M, N, K, act, dtype: lib.rxmet_linear_int8(
        p, K, p, p, K, p, None, None, 0, p, M, N, K, act, dtype, None, None)
    says(lin(1, 1, 131072, 0, 0), "K between 1 and 131071")
    says(lin(1, 1, 8, 4, 0), "activation")
    says(lin(1, 1, 8, 0, 3), "fp32, fp16 or bf16")
    assert lin(0, 1, 8, 0, 0) == 0

    def cache(dim=64, page=16, heads=2, pages=4):
        return rxmet_lib.KvCache(p, p, p, p, pages, heads, page, dim, 0)

    table = rxmet_lib.KvTable(p, 1, 1, 1)
    att = lambda c, heads, dtype=1: lib.rxmet_kv_attention(
        ctypes.byref(c), ctypes.byref(table), p, None, 1, 1, 1, p, 64, 64, heads, 1.0, 1, 0, p,
        dtype, None, None)
    says(att(cache(dim=80), 2), "head dimension")
    says(att(cache(page=48), 2), "page size")
    says(att(cache(), 3), "multiple")
    says(att(cache(), 2, 0), "fp16 or bf16")
    big = rxmet_lib.KvTable(p, 1, 65536, 1)
    says(lib.rxmet_kv_append(ctypes.byref(cache()), ctypes.byref(big), p, None, 65536, 1, p, 64, 64,
                             p, 64, 64, 0, None), "65535 sequences")
    says(lib.rxmet_kv_append(ctypes.byref(cache()), ctypes.byref(table), p, None, 2, 1, p, 64, 64, p,
                             64, 64, 0, None), "one token a sequence")
