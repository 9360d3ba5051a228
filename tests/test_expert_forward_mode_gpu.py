"""Forward-mode derivatives of the expert operators, which have none: asked for, they raise on both routes to
the kernels and never go missing."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import expert_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["logits", "y", "weights", "residual"])
def test_dual_tensors_are_refused(cuda, monkeypatch, native, grad, which):
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    x = torch.randn(20, 8, device=cuda)
    ids, w = ops.route_experts(x, 3)
    g = ops.group_experts(ids, 8)
    y, r = torch.randn(60, 32, device=cuda), torch.randn(20, 32, device=cuda)
    args = dict(logits=x, y=y, weights=w, residual=r)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="(?i)jvp|forward"):
            if which == "logits":
                ops.route_experts(args["logits"], 3)
            else:
                ops.experts_combine(args["y"], args["weights"], g, residual=args["residual"])


def test_a_dual_level_alone_changes_nothing(cuda):
    x = torch.randn(20, 8, device=cuda)
    want = ops.route_experts(x, 3)
    with fwd.dual_level():
        got = ops.route_experts(x, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
