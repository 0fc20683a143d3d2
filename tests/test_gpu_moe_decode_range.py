"""moe.moe_decode where its inner values need all their digits or come near the largest ones, next to the others in
tests/test_gpu_moe_decode.py."""
import math

import pytest
import torch

from cinnamon_amd import kernels, layers, moe
from tests.test_gpu_moe_decode import DT, E4M3, STEP, U, check, definition, inputs


def pairs(dev, T, D, dt, wt, lead, gen):
    """x and an expert whose channels i and i + D differ by 2^-13 or so of their h, and whose i-th output is the
    difference of these two.  Only x's first two channels count; weights have four bits and scales are one."""
    H = 2 * D
    w12 = torch.zeros(2, 2, D, D)  # W1 and W2, the first and the second of a pair
    w12[0, :, :, 0] = torch.randint(8, 16, (D,), generator=gen) / 8
    w12[1, :, :, 0] = torch.randint(8, 16, (D,), generator=gen) / 8
    w12[1, 0, :, 1], w12[1, 1, :, 1] = 1.125, 1.0
    w3 = torch.cat([torch.eye(D), -torch.eye(D)], 1)
    x = torch.zeros(T, D)
    x[:, 0] = 0.5 + torch.rand(T, generator=gen)
    x[:, 1] = 2.0 ** -10 * (1 + torch.rand(T, generator=gen))
    w12, w3 = w12.view(2 * H, D).expand(*lead, -1, -1), w3.expand(*lead, -1, -1)
    x = x.to(DT[dt]).to(dev)
    if wt == "bf16":
        return x, (w12.bfloat16().contiguous().to(dev), None, w3.bfloat16().contiguous().to(dev), None)
    ones = lambda r, c: torch.ones(*lead, -(-r // 128), -(-c // 128), device=dev)  # noqa: E731
    return x, (w12.contiguous().to(E4M3).to(dev), ones(2 * H, D), w3.contiguous().to(E4M3).to(dev), ones(D, H))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("wt", ["fp8", "bf16"])
@pytest.mark.parametrize("where", ["routed", "shared"])
@pytest.mark.parametrize("T", [1, 16, 20, 100])
def test_h_keeps_24_bits(dev, T, dt, wt, where):
    """h is within 24 u of its value (W1 x and W2 x: two terms and a scale, 4 u each, the first 1.3 times through silu;
    silu's exponential, sum and quotient 8 u; three products 4 u) and its parts within u more; the output is the
    difference of two h: 4 u of each for the units' sum, and one rounding of a result 2^-13 as large."""
    D = 128
    gen = torch.Generator().manual_seed(T)
    lead = (1,) if where == "routed" else ()
    x, w = pairs(dev, T, D, dt, wt, lead, gen)
    r = torch.zeros(1, D, device=dev)
    if where == "routed":
        got, _, weights = moe.moe_decode(x, r, w, 1, return_routing=True)
        weight = weights.double()
    else:
        none = pairs(dev, T, D, dt, wt, (1,), gen)[1]
        none[2].zero_()
        got, weight = moe.moe_decode(x, r, none, 1, shared=w), 1.0
    w12, w3 = (v.reshape(v.shape[-2:]).float().double() for v in (w[0], w[2]))
    a, b = (x.double() @ w12.t()).chunk(2, -1)
    h = weight * a * torch.sigmoid(a) * b
    want, size = h @ w3.t(), h.abs() @ w3.abs().t()
    assert (want.abs() < 2.0 ** -11 * size).all() and (want != 0).all()
    tol = (24 + 1 + 4) * U * size + (1 + 2.0 ** -8) * STEP[got.dtype] * want.abs() + 2.0 ** -25
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), ((got.double() - want).abs() / tol)[bad].max()


LARGEST = torch.finfo(torch.float32).max
LARGEST16 = 2.0 ** 128 - 2.0 ** 120  # of bf16
FAR = 2.0 ** 128 - 2.0 ** 119  # from here on rounding to bf16 gives infinity


@pytest.mark.gpu
@pytest.mark.parametrize("wt", ["fp8", "bf16"])
@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("big", [LARGEST16, FAR - 2.0 ** 104, FAR, -FAR, LARGEST, -LARGEST])
def test_states_next_to_the_largest(dev, big, T, wt):
    """Finite fp32 states whose rounding to bf16 is infinite: their weights are zero, or (bf16 weights) bring them
    back to the others' size."""
    D, H, E = 144, 64, 2
    x, r, experts, shared = inputs(dev, T, D, H, E, "fp32", wt, H)
    r[:, 3] = 0
    for w in (experts, shared):
        w[0].view(torch.uint8 if wt == "fp8" else w[0].dtype)[..., 3] = 0
        if wt == "bf16":
            w[0][..., 3] = 2.0 ** -126 * torch.randint(-2, 3, w[0].shape[:-1], generator=torch.Generator().manual_seed(4)).to(dev)
    x[T - 1, 3] = big
    got = moe.moe_decode(x, r, experts, 2, shared=shared, return_routing=True)
    assert torch.isfinite(got[0]).all()
    check(got, definition(x, r, experts, 2, shared=shared))
    x[T - 1, 3] = math.copysign(math.inf, big)
    assert not torch.isfinite(moe.moe_decode(x, r, experts, 2, shared=shared)[T - 1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 20, 100])
@pytest.mark.parametrize("sign", [1, -1])
def test_h_next_to_the_largest(dev, T, dt, sign):
    """h = 2^64 (2^64 - 2^56 + 2^55 v), v in [1, 2): finite, rounding to infinity in bf16.  Its three products and one sum
    are within 8 u (silu of 2^64 is exact), its parts and the output's product within 4 u more."""
    D, H = 64, 32
    x = torch.zeros(T, D, device=dev)
    x[:, 0] = 1
    x[:, 1] = 1 + torch.arange(T, device=dev) / 128
    x = x.to(DT[dt])
    w12, w3 = torch.zeros(1, 2 * H, D, device=dev), torch.zeros(1, D, H, device=dev)
    w12[:, 0, 0] = 2.0 ** 64
    w12[:, H, 0], w12[:, H, 1] = sign * (2.0 ** 64 - 2.0 ** 56), sign * 2.0 ** 55
    w3[:, :, 0] = 2.0 ** -120
    r = torch.zeros(1, D, device=dev)
    got = moe.moe_decode(x, r, (w12.bfloat16(), None, w3.bfloat16(), None), 1)
    want = sign * 2.0 ** -56 * (2.0 ** 64 - 2.0 ** 56 + 2.0 ** 55 * x[:, 1:2].double()).expand(T, D)
    assert (want.abs() * 2.0 ** 120 >= FAR).all() and (want.abs() * 2.0 ** 120 <= LARGEST).all()
    assert ((got.double() - want).abs() <= (12 * U + (1 + 2.0 ** -8) * STEP[got.dtype]) * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("wt", ["fp8", "bf16"])
def test_whatever_requires_a_gradient_has_its_backward_refused(dev, wt):
    """One tensor of the call at a time; the result is that of the call without."""
    x, r, experts, shared = inputs(dev, 3, 256, 128, 4, "bf16", wt, 128)
    bias = torch.zeros(4, device=dev)

    def call(x, r, bias, *w):
        return moe.moe_decode(x, r, w[:4], 2, bias=bias, shared=w[4:], return_routing=True)

    tensors = [x, r, bias, *experts, *shared]
    want = call(*tensors)
    assert not want[0].requires_grad
    for i, t in enumerate(tensors):
        if t is None or t.dtype == E4M3:
            continue
        for leaf in (t.clone().requires_grad_(), torch.nn.Parameter(t.clone())):
            args = [leaf if j == i else v for j, v in enumerate(tensors)]
            got = call(*args)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            with pytest.raises(RuntimeError, match="autograd"):
                got[0].sum().backward()
            with torch.no_grad():
                got = call(*args)
            assert not got[0].requires_grad and torch.equal(got[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("cached", [False, True])
def test_trainable_experts_have_their_backward_refused(dev, cached):
    torch.manual_seed(5)
    experts = layers.GroupedExperts(4, 256, 128).to(dev)
    x, r = torch.randn(3, 256, device=dev).bfloat16(), torch.randn(4, 256, device=dev)
    if cached:
        kernels.set_weight_cache(experts)
    with torch.no_grad():
        want = moe.moe_decode(x, r, experts, 2)
    assert not want.requires_grad
    for frozen in ((), ("w12",), ("w3",)):
        for name in ("w12", "w3"):
            getattr(experts, name).requires_grad_(name not in frozen)
        out = moe.moe_decode(x, r, experts, 2)
        assert torch.equal(out, want)
        with pytest.raises(RuntimeError, match="autograd"):
            out.sum().backward()
    experts.requires_grad_(False)
    out = moe.moe_decode(x, r, experts, 2)
    assert not out.requires_grad and torch.equal(out, want)
