"""No operator has a forward-mode derivative: an input or a gradient that carries one is refused, never computed without it.
The launches are replaced, so that these run on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

from cinnamon_amd import kernels, lm_head, moe, norm, rotary


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


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a device, for the public functions' checks."""
    is_cuda = True


def on_device(t):
    return t.as_subclass(OnDevice)


def test_differentiable_operators_refuse_tangents(monkeypatch):
    """moe_gate, apply_rotary, linear_cross_entropy and indexer_scores_fp8 (its weights), at the call and in the backward."""
    logits, x, y = on_device(torch.randn(3, 8)), torch.randn(1, 3, 2, 32), torch.zeros(3, dtype=torch.int64)
    cos = on_device(torch.ones(3, 16))
    calls = [(logits, lambda t: moe.moe_gate(t, 2)[1]), (on_device(x), lambda t: rotary.apply_rotary(t, cos, cos)),
             (on_device(x), lambda t: rotary.apply_rotary(on_device(x), cos, cos, k=t)[1]),
             (logits, lambda t: lm_head.linear_cross_entropy(t, on_device(torch.randn(5, 8)), on_device(y))),
             (logits, lambda t: lm_head.linear_cross_entropy(on_device(torch.randn(3, 8)), t, on_device(y))),
             (on_device(torch.randn(1, 3, 2)), lambda t: kernels.indexer_scores_fp8(on_device(x), on_device(x[:, :, 0]), t, 1.0))]
    for t, f in calls:
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            f(forward_ad.make_dual(t, torch.ones_like(t)))
    for module, name in ((moe, "_launch_gate_backward"), (rotary, "_launch"), (lm_head, "_launch_backward"), (kernels, "_launch_wgrad")):
        monkeypatch.setattr(module, name, lambda *a: pytest.fail("launched"))

    class Ctx:
        saved_tensors, options, needs_input_grad, softmax_scale, with_k, save_q = (X, X, X, X), (0,) * 8, (True,) * 8, 1.0, False, True

    with forward_ad.dual_level():
        g = forward_ad.make_dual(X, X)
        for f in (lambda: moe._gate_gradient(Ctx, None, g, None), lambda: rotary._rotary_turn_back(Ctx, g, None),
                  lambda: lm_head._gradients(Ctx, g), lambda: kernels._IndexerScoresQ.backward(Ctx, g),
                  lambda: kernels._indexer_backward(Ctx, g), lambda: kernels._indexer_q_backward(Ctx, g, None, None)):
            with pytest.raises(NotImplementedError):
                f()
