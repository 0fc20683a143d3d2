"""moe.moe_decode where its inner values need all their digits, next to the others in tests/test_gpu_moe_decode.py."""
import pytest
import torch

from cinnamon_amd import moe

U = 2.0 ** -24
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


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
