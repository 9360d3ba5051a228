"""Leading axes, single tokens without one, and broadcast inputs of the routing and the rows' sum: the same results
and gradients as rows have."""
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu

LEADS = [(), (1,), (24,), (2, 3, 4), (4, 1, 6)]


def flat(t, keep=1):
    return t.reshape(-1, *t.shape[t.dim() - keep:])


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("lead", LEADS)
def test_leading_axes(cuda, monkeypatch, native, lead):
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    gen = torch.Generator(cuda).manual_seed(len(lead))
    rand = lambda *s: torch.randn(*s, device=cuda, generator=gen)
    x = rand(*lead, 16).requires_grad_()
    n = x.numel() // 16
    y, r, d = rand(n * 3, 70).requires_grad_(), rand(*lead, 70).requires_grad_(), rand(*lead, 70)

    def run(x, r, d):
        ids, w = ops.route_experts(x, 3)
        g = ops.group_experts(ids, 16)
        out = ops.experts_combine(y, w, g, residual=r)
        return ids, w, g.places, out, torch.autograd.grad(out, (x, y, r), d)

    ids, w, places, out, (dx, dy, dr) = run(x, r, d)
    assert ids.shape == w.shape == places.shape == (*lead, 3) and out.shape == (*lead, 70)
    assert dx.shape == x.shape and dy.shape == y.shape and dr.shape == r.shape
    x2, r2 = flat(x.detach()).requires_grad_(), flat(r.detach()).requires_grad_()
    ids2, w2, places2, out2, (dx2, dy2, dr2) = run(x2, r2, flat(d))
    for a, b in ((ids, ids2), (w, w2), (places, places2), (out, out2), (dx, dx2), (dr, dr2)):
        assert torch.equal(flat(a), b)
    assert torch.equal(dy, dy2)


@pytest.mark.parametrize("native", [True, False])
def test_broadcast_inputs(cuda, monkeypatch, native):
    """One row for all tokens: its gradient is the sum of theirs."""
    if not native:
        monkeypatch.setattr(ops, "_ext", False)
    T, k, N = 40, 3, 33
    gen = torch.Generator(cuda).manual_seed(2)
    rand = lambda *s: torch.randn(*s, device=cuda, generator=gen)
    one, g = rand(1, 16).requires_grad_(), rand(T, k)
    ids, w = ops.route_experts(one.expand(T, 16), k, renormalize=False)
    (d,) = torch.autograd.grad(w, one, g)
    every = one.detach().expand(T, 16).contiguous().requires_grad_()
    ids2, w2 = ops.route_experts(every, k, renormalize=False)
    (d2,) = torch.autograd.grad(w2, every, g)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    torch.testing.assert_close(d, d2.sum(0, keepdim=True), rtol=0, atol=T * 2.0 ** -24 * float(d2.abs().sum(0).max()))
    groups = ops.group_experts(torch.randint(0, 5, (T, k), dtype=torch.int32, device=cuda, generator=gen), 5)
    y, wt, r, do = rand(1, N), rand(1, k), rand(1, N), rand(T, N)
    small = [t.requires_grad_() for t in (y, wt, r)]
    large = [t.detach().expand(n, -1).contiguous().requires_grad_() for t, n in zip(small, (T * k, T, T))]
    a = ops.experts_combine(y.expand(T * k, N), wt.expand(T, k), groups, residual=r.expand(T, N))
    b = ops.experts_combine(large[0], large[1], groups, residual=large[2])
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, small, do), torch.autograd.grad(b, large, do)):
        # sums of as many numbers in another order: each partial sum within a half step
        torch.testing.assert_close(p, q.sum(0, keepdim=True), rtol=0,
                                   atol=T * k * 2.0 ** -24 * float(q.abs().sum(0).max()))
