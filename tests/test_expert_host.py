"""The expert layers' operators without a GPU: their oracle against itself, and what they refuse."""
import ctypes

import numpy as np
import pytest
import torch

import expert_ops as ops
import expert_oracle as O
import rxmet_lib


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_oracle_route_gradient_is_the_weights_derivative(score, renormalize):
    rng = np.random.default_rng(3)
    x, g = rng.standard_normal((4, 12)), rng.standard_normal((4, 3))
    ids = O.choose(x, 3, score)
    f = lambda v: (O.weights(v, ids, score, renormalize, 1.5) * g).sum()
    dx = O.route_backward(x, ids, g, score, renormalize, 1.5)
    for _ in range(5):
        a, t = rng.standard_normal(x.shape), 1e-5
        assert abs((f(x + t * a) - f(x - t * a)) / (2 * t) - (dx * a).sum()) < 1e-7


def test_oracle_combine_gradient_is_the_sums_derivative():
    rng = np.random.default_rng(4)
    ids = rng.integers(-1, 4, (5, 2)).astype(np.int32)
    _, _, places = O.group(ids, 4)
    y, w, g = rng.standard_normal((10, 7)), rng.standard_normal((5, 2)), rng.standard_normal((5, 7))
    dy, dw, _ = O.combine_backward(y, w, places, g)
    f = lambda y, w: (O.combine(y, w, places, None)[0] * g).sum()
    a, b, t = rng.standard_normal(y.shape), rng.standard_normal(w.shape), 1e-5
    assert abs((f(y + t * a, w + t * b) - f(y - t * a, w - t * b)) / (2 * t) - (dy * a).sum()
               - (dw * b).sum()) < 1e-7


def test_oracle_sees_a_planted_mistake():
    """The comparisons of the GPU tests fail where a tie goes to the later expert or a sum leaves a row out."""
    x = np.array([[0.0, 1.0, 1.0, 0.5]])
    assert O.choose(x, 2).tolist() == [[1, 2]]
    assert O.choose(x[:, ::-1], 1).tolist() != [[2]]
    rng = np.random.default_rng(5)
    y, w = rng.standard_normal((4, 9)), np.full((2, 2), 0.5)
    places = np.arange(4).reshape(2, 2)
    out, _ = O.combine(y, w, places, None)
    places[0, 1] = -1
    assert np.abs(O.combine(y, w, places, None)[0] - out).max() > 1e-2


def test_oracle_groups():
    offsets, entries, places = O.group(np.array([[2, 0], [-1, 2], [0, 7]]), 3)
    assert offsets.tolist() == [0, 2, 2, 4] and entries.tolist() == [1, 4, 0, 3, 2, 5]
    assert places.tolist() == [[2, 0], [-1, 3], [1, -1]]


def test_oracle_choice_by_groups_and_bias():
    x = np.array([[3.0, 0.0, 2.0, 1.9, 1.0, 0.9]])
    # by the best of a group 0 and 1, by the best two 1 and 0 or 2
    assert O.choose(x, 2, "sigmoid", None, 3, 1, 1).tolist() == [[0, 1]]
    assert O.choose(x, 2, "sigmoid", None, 3, 1, 2).tolist() == [[2, 3]]
    assert O.choose(x, 1, "sigmoid", np.array([0, 0, 0, 0, 0, 1.0])).tolist() == [[5]]
    assert O.choose(np.array([[np.nan, -np.inf, 0.0]]), 3).tolist() == [[2, 0, 1]]


def test_operators_refuse_host_tensors():
    x = torch.zeros(3, 4)
    ids = torch.zeros(3, 2, dtype=torch.int32)
    g = ops.ExpertGroups(torch.zeros(5, dtype=torch.int32), torch.zeros(6, dtype=torch.int32), ids)
    for f in (lambda: ops.route_experts(x, 2), lambda: ops.group_experts(ids, 4),
              lambda: ops.experts_linear_int8(x.to(torch.int8), x[:, 0], x.to(torch.int8)[None], x, g),
              lambda: ops.experts_combine(torch.zeros(6, 4), torch.zeros(3, 2), g)):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f()


@pytest.mark.parametrize("what, match", [
    (dict(score="tanh"), "score must be"), (dict(groups=3), "groups must be"),
    (dict(groups=4, top_groups=5), "top_groups"), (dict(group_best=3), "group_best"),
    (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"), (dict(groups=4, top_groups=1, top_k=3), "top_k"),
    (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(experts=100, top_k=65), "top_k")])
def test_routers_that_are_refused(what, match):
    args = dict(experts=8, top_k=2, score="softmax", groups=1, top_groups=None, group_best=1,
                renormalize=True, scale=1.0)
    ops._router(**args)
    with pytest.raises(RuntimeError, match=match):
        ops._router(**{**args, **what})


def test_library_refuses_before_any_device_call():
    lib = rxmet_lib.load()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf) // 16 * 16 + 16

    def says(rc, text):
        assert rc == -22 and text in lib.rxmet_last_error().decode(), lib.rxmet_last_error()

    def route(tokens=1, dtype=0, **kw):
        r = rxmet_lib.Router(**{**dict(experts=8, top_k=2, score=0, renormalize=1, groups=1,
                                       top_groups=1, group_best=1, scale=1.0), **kw})
        return (lib.rxmet_route_forward(ctypes.byref(r), p, 8, None, p, p, tokens, dtype, None),
                lib.rxmet_route_backward(ctypes.byref(r), p, 8, p, p, p, tokens, dtype, None))[::-1][0]

    says(route(experts=1025), "1 to 1024 experts")
    says(route(experts=0), "1 to 1024 experts")
    says(route(score=2), "unknown score")
    says(route(groups=3), "equal length")
    says(route(groups=0), "equal length")
    says(route(top_groups=2), "top_groups")
    says(route(group_best=0), "group_best")
    says(route(top_k=9), "top_k")
    says(route(dtype=3), "fp32, fp16 or bf16")
    says(route(tokens=-1), "tokens")
    assert route(tokens=0) == 0

    group = lambda n, e, ws=None: lib.rxmet_group_experts(p, n, e, p, p, p, ws, None)
    says(group(1, 1025), "1 to 1024 experts")
    says(group((1 << 26) + 1, 8), "2^26 entries")
    says(group(1 << 20, 8), "workspace")
    assert lib.rxmet_group_experts_workspace_bytes(16, 8) == 0
    assert lib.rxmet_group_experts_workspace_bytes(1 << 20, 8) > 0

    def groups(tokens=1, top_k=2, experts=4):
        return ctypes.byref(rxmet_lib.ExpertGroups(p, p, p, tokens, top_k, experts))

    lin = lambda g, N=8, K=16, act=0, dtype=0: lib.rxmet_experts_linear_int8(
        g, 0, p, K, p, p, K, K * N, p, None, p, N, K, 0, act, dtype, None)
    says(lin(groups(top_k=65)), "top_k")
    says(lin(groups(experts=0)), "1 to 1024 experts")
    says(lin(groups(), K=131072), "K between 1 and 131071")
    says(lin(groups(), N=0), "N must be between")
    says(lin(groups(), act=4), "activation")
    says(lin(groups(), dtype=3), "fp32, fp16 or bf16")
    says(lin(groups(tokens=1 << 24, top_k=64)), "too many outputs")
    assert lin(groups(tokens=0)) == 0

    comb = lambda g, N=8, dtype=0: lib.rxmet_experts_combine(g, p, N, p, None, 0, p, N, dtype, None)
    says(comb(groups(tokens=-1)), "tokens")
    says(comb(groups(), N=0), "N must be between")
    says(comb(groups(), dtype=3), "fp32, fp16 or bf16")
    assert comb(groups(tokens=0)) == 0
    back = lambda dy, dw, y: lib.rxmet_experts_combine_backward(groups(), p, 8, y, 8, p, dy, dw, 8, 0, None)
    says(back(None, p, None), "needs y")
    assert back(None, None, None) == 0
