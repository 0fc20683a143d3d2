"""No operator has a forward-mode derivative: an input or a gradient that carries one is refused, never computed without it.
The launches are replaced, so that these run on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

from cinnamon_amd import kernels, norm


@pytest.fixture
def launches(monkeypatch):
    """norm's launches in elementary operations, whose own tangents would show, and its checks off."""
    def forward(y, residual, weight, post_weight, gate, scale, value, eps, train=True):
        y = y.detach()
        return y * 2, None if residual is None else residual.detach() * 3, y.new_zeros(2 * (y.numel() // y.shape[-1]))

    def backward(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs):
        return [torch.ones_like(t) if need and t is not None else None
                for t, need in zip((y, residual, weight, post_weight, gate, scale), needs)]

    monkeypatch.setattr(norm, "_check", lambda *a: None)
    monkeypatch.setattr(norm, "_launch", forward)
    monkeypatch.setattr(norm, "_launch_backward", backward)


X, W = torch.arange(12.0).view(3, 4), torch.ones(4)
CALLS = {"rms_norm": lambda x: norm.rms_norm(x, W), "weight": lambda x: norm.rms_norm(X, x[0]),
         "residual": lambda x: norm.block_norm(X, x, W)[1], "gate": lambda x: norm.block_norm(X, X, gate=x)[0],
         "scale": lambda x: norm.block_norm(X, X, residual_scale=x[0, 0])[1]}


@pytest.mark.parametrize("name", CALLS)
def test_norms_refuse_tangents(launches, name):
    f = CALLS[name]
    f(X)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(f, (X,), (X,))
    with pytest.raises(NotImplementedError):
        torch.func.jacfwd(f)(X)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.hessian(lambda x: f(x).sum())(X)
    with forward_ad.dual_level():
        f(X)  # no tangent
        with pytest.raises(NotImplementedError):
            f(forward_ad.make_dual(X, X))
        with pytest.raises(NotImplementedError):
            f(forward_ad.make_dual(X.clone().requires_grad_(), X))


def test_norms_among_tangents_of_others(launches):
    def f(x):
        return norm.rms_norm(X * 2, W) + x

    out, tangent = torch.func.jvp(f, (X,), (W.expand(3, 4),))
    assert torch.equal(out, X * 4 + X) and torch.equal(tangent, W.expand(3, 4))


def test_norms_refuse_tangents_of_gradients(launches):
    for op in (False, True):
        leaf = X.clone().requires_grad_()
        n, _ = norm.block_norm(leaf, X, W) if not op else norm._norm_op(leaf, X, W, None, None, None, 1.0, 1e-6)[:2]
        torch.autograd.grad(n, leaf, X, retain_graph=True)
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(n, leaf, forward_ad.make_dual(X, X))


def test_operators_without_a_gradient_refuse_tangents():
    """moe.moe_decode and the routed path's parts."""
    @kernels.custom_op("test_refuses_tangents", "(Tensor x) -> Tensor")
    def op(x):
        return x.clone()

    assert torch.equal(kernels._run_detached(op, X), X)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: kernels._run_detached(op, x), (X,), (X,))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        kernels._run_detached(op, forward_ad.make_dual(X, X))
