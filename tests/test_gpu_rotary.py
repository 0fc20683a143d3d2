"""rotary.apply_rotary and rotary_tables against their definition in 64 bits (GPU for the
operator, CPU for the tables and the refusals).

A turned value is a sum of two fp32 products: with x0, x1 the pair and m the tables' largest
factor, within 3 u m (|x0| + |x1|), u = 2^-24, before its one rounding to the output's type.
"""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, rotary

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
LEAST = {"bf16": 1e-37, "fp16": 2.0 ** -24, "fp32": 1e-37}


def turn(x, cos, sin, positions, interleaved, start, inverse=False):
    """(result, magnitude of each value's pair) of x [B, L, H, D] in 64 bits."""
    x = x.detach().double().cpu()
    B, L = x.shape[:2]
    P, half = cos.shape
    p = torch.arange(L).expand(B, L) if positions is None else positions.cpu().expand(B, L)
    c = torch.where((p < 0)[..., None], 1.0, cos.cpu().double()[p.clamp(0, P - 1)])
    s = torch.where((p < 0)[..., None], 0.0, sin.cpu().double()[p.clamp(0, P - 1)])
    c, s = (torch.where((p >= P)[..., None], math.nan, t).unsqueeze(2) for t in (c, s))
    if inverse:
        s = -s
    i = torch.arange(half)
    i0, i1 = (start + 2 * i, start + 2 * i + 1) if interleaved else (start + i, start + half + i)
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    mag[..., i0] = mag[..., i1] = x[..., i0].abs() + x[..., i1].abs()
    return y, mag


def check(got, ref, dt, most=1.0):
    y, mag = ref
    g = got.detach().double().cpu()
    assert got.dtype == DT[dt] and got.shape == y.shape
    assert torch.equal(torch.isnan(g), torch.isnan(y))
    tol = STEP[dt] * y.abs() + 3 * U * most * mag * (1 + STEP[dt]) + LEAST[dt]
    d = (g - y).abs()
    ok = (d <= tol) | torch.isnan(y)
    assert ok.all(), d[~ok].max()
    copied = mag == 0
    assert torch.equal(g[copied & ~torch.isnan(y)], y[copied & ~torch.isnan(y)])


CASES = [
    # B, L, H, Hk, D, start, rot, interleaved, positions, dtype
    (1, 1, 1, 1, 2, 0, 2, True, "none", "fp32"),
    (64, 1, 16, 1, 128, 64, 64, True, "each", "bf16"),
    (3, 1, 5, 2, 130, 2, 64, False, "each", "bf16"),
    (2, 100, 16, 1, 64, 0, 64, True, "none", "bf16"),
    (2, 33, 3, 3, 192, 128, 64, False, "far", "fp16"),
    (1, 257, 4, 4, 96, 16, 32, False, "each", "fp32"),
    (3, 17, 2, 1, 65, 0, 64, True, "none", "bf16"),
    (2, 29, 3, 1, 97, 1, 64, False, "far", "fp16"),
    (2, 31, 4, 2, 100, 8, 6, True, "each", "fp32"),
    (2, 31, 4, 2, 100, 8, 6, False, "each", "bf16"),
    (1, 7, 40, 8, 256, 0, 256, False, "none", "fp16"),
    (5, 1023, 2, 1, 128, 0, 16, True, "far", "bf16"),
]


def inputs(case, dev, seed=1):
    B, L, H, Hk, D, start, rot, inter, pos, dt = case
    g = torch.Generator().manual_seed(seed)
    q, k, gq, gk = (torch.randn(B, L, h, D, generator=g).to(DT[dt]).to(dev) for h in (H, Hk, H, Hk))
    P = 2 * L + 50
    cos, sin = rotary.rotary_tables(rot, P, device=dev)
    p = {"none": None, "far": torch.arange(L) + P - L, "each": torch.randint(0, P, (B, L), generator=g)}[pos]
    return q, k, gq, gk, cos, sin, p if p is None else p.to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rotary_forward_and_backward(dev, case):
    start, inter, dt = case[5], case[7], case[9]
    q, k, gq, gk, cos, sin, p = inputs(case, dev)
    kw = dict(positions=p, interleaved=inter, start=start)
    oq, ok = rotary.apply_rotary(q, cos, sin, k=k, **kw)
    check(oq, turn(q, cos, sin, p, inter, start), dt)
    check(ok, turn(k, cos, sin, p, inter, start), dt)
    alone = rotary.apply_rotary(q, cos, sin, **kw)
    assert torch.equal(alone, oq)
    ql, kl = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    o = rotary.apply_rotary(ql, cos, sin, k=kl, **kw)
    dq, dk = torch.autograd.grad(o, [ql, kl], [gq, gk])
    check(dq, turn(gq, cos, sin, p, inter, start, True), dt)
    check(dk, turn(gk, cos, sin, p, inter, start, True), dt)
    # one gradient alone, through either
    (dk2,) = torch.autograd.grad(rotary.apply_rotary(q, cos, sin, k=kl, **kw)[1], [kl], gk)
    (dq2,) = torch.autograd.grad(rotary.apply_rotary(ql, cos, sin, k=kl, **kw)[0], [ql], gq)
    assert torch.equal(dk2, dk) and torch.equal(dq2, dq)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_rotary_strides(dev, inter, dt):
    g = torch.Generator().manual_seed(2)
    B, L, H, D = 2, 37, 4, 64
    cos, sin = rotary.rotary_tables(32, 200, device=dev)
    fused = torch.randn(B, L, 3 * H * D + 8, generator=g).to(DT[dt]).to(dev)
    heads_first = torch.randn(B, H, L, D, generator=g).to(DT[dt]).to(dev)
    odd = torch.randn(B, L, H, D + 1, generator=g).to(DT[dt]).to(dev)
    other = torch.randn(B, L, D, H, generator=g).to(DT[dt]).to(dev)
    views = [fused[..., H * D:2 * H * D].unflatten(-1, (H, D)), heads_first.transpose(1, 2), odd[..., 1:], odd[..., :D],
             other.transpose(2, 3), fused[:, :, 4:4 + D].unsqueeze(2).expand(B, L, H, D),
             torch.randn(B, 2 * L, H, D, generator=g).to(DT[dt]).to(dev)[:, ::2]]
    p = torch.randint(0, 200, (2 * L, B), generator=g).to(dev).t()[:, ::2]  # strided positions
    for v in views:
        got = rotary.apply_rotary(v, cos, sin, positions=p, interleaved=inter, start=16)
        check(got, turn(v, cos, sin, p, inter, 16), dt)
        leaf = v.detach().requires_grad_(True)
        o = rotary.apply_rotary(leaf, cos, sin, positions=p, interleaved=inter, start=16)
        (d,) = torch.autograd.grad(o.sum(), [leaf])  # an expanded gradient
        check(d, turn(torch.ones(B, L, H, D), cos, sin, p, inter, 16, True), dt)
    # tables that are views, and [B, L, D] with no head dimension
    wide = torch.stack([cos, sin], -1)
    assert torch.equal(rotary.apply_rotary(views[0], wide[..., 0], wide[..., 1], interleaved=inter),
                       rotary.apply_rotary(views[0], cos, sin, interleaved=inter))
    x3 = fused[..., :D]
    a, b = rotary.apply_rotary(views[0], cos, sin, k=x3, interleaved=inter)
    assert b.shape == x3.shape and torch.equal(b, rotary.apply_rotary(x3.unsqueeze(2), cos, sin, interleaved=inter)[:, :, 0])
    assert torch.equal(a, rotary.apply_rotary(views[0], cos, sin, interleaved=inter))
    for dtype in (torch.int32, torch.int16, torch.uint8):
        assert torch.equal(rotary.apply_rotary(x3, cos, sin, positions=p.to(dtype), interleaved=inter),
                           rotary.apply_rotary(x3, cos, sin, positions=p, interleaved=inter))


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_rotary_padding_and_positions_past_the_table(dev, inter, dt):
    g = torch.Generator().manual_seed(3)
    cos, sin = rotary.rotary_tables(32, 10, device=dev)
    x = torch.randn(2, 6, 2, 48, generator=g).to(DT[dt]).to(dev)
    p = torch.tensor([[0, 9, 10, -1, 2 ** 40, 3], [-(2 ** 62), -1, -1, 9, 1, 2 ** 62]], device=dev)
    got = rotary.apply_rotary(x, cos, sin, positions=p, interleaved=inter, start=8)
    check(got, turn(x, cos, sin, p, inter, 8), dt)
    assert torch.isnan(got[0, 2, :, 8:40]).all() and torch.equal(got[0, 2, :, :8], x[0, 2, :, :8])
    assert torch.equal(got[0, 3], x[0, 3])


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,start,rot", [(48, 8, 32), (33, 3, 6), (64, 0, 64)])
def test_rotary_padding_may_hold_anything(dev, inter, dt, D, start, rot):
    """A token at a negative position keeps its bits, infinities, NaN and the zeros' signs among them,
    and so does its gradient."""
    g = torch.Generator().manual_seed(4)
    cos, sin = rotary.rotary_tables(rot, 10, device=dev)
    x = torch.randn(2, 6, 3, D, generator=g).to(DT[dt])
    odd = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 1.0, torch.finfo(DT[dt]).max, 1e-30]).to(DT[dt])
    x[:, ::2] = odd[torch.randint(0, len(odd), x[:, ::2].shape, generator=g)]
    x = x.to(dev)
    p = torch.tensor([[-1, 9, -7, 3, -(2 ** 40), 0], [-1, -1, -2, 5, -(2 ** 62), 2]], device=dev)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    for k in (None, x[:, :, :1]):
        leaf = x.clone().requires_grad_(True)
        out = rotary.apply_rotary(leaf, cos, sin, k=k, positions=p, interleaved=inter, start=start)
        got = out if k is None else out[0]
        (d,) = torch.autograd.grad(got, [leaf], x)
        for y in (got.detach(), d):
            assert torch.equal(y[p < 0].view(bits), x[p < 0].view(bits))
        if k is not None:
            assert torch.equal(out[1][p < 0].view(bits), x[:, :, :1][p < 0].view(bits))
    rest = (p >= 0) & torch.isfinite(x.float()).all(-1).all(-1)
    y, mag = turn(torch.where(rest[..., None, None], x, 0), cos, sin, p, inter, start)
    rest = rest.cpu()
    check(got.detach().cpu()[rest], (y[rest], mag[rest]), dt)


@pytest.mark.gpu
def test_rotary_empty(dev):
    cos, sin = rotary.rotary_tables(32, 10, device=dev)
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)):
        x = torch.empty(shape, device=dev, requires_grad=True)
        o = rotary.apply_rotary(x, cos, sin)
        assert o.shape == shape
        assert torch.autograd.grad(o.sum(), [x])[0].shape == shape
    none = torch.empty(0, 16, device=dev)
    assert rotary.apply_rotary(torch.empty(1, 0, 2, 64, device=dev), none, none).numel() == 0
    p = torch.tensor([3, -1], device=dev)
    y = rotary.apply_rotary(torch.ones(1, 2, 1, 32, device=dev), none, none, positions=p)
    assert torch.isnan(y[0, 0]).all() and (y[0, 1] == 1).all()


@pytest.mark.gpu
def test_rotary_offsets_past_32_bits(dev):
    """The last tokens of a bf16 tensor of more than 2^32 bytes, read and written in place of views."""
    cos, sin = rotary.rotary_tables(64, 1 << 20, device=dev)
    L, H, D = 1 << 20, 18, 128
    x = torch.empty(1, L, H, D, dtype=torch.bfloat16, device=dev)
    x[:, -3:] = 1.5
    x[:, :3] = -2.0
    y = rotary.apply_rotary(x, cos, sin, start=64)
    for sl in (slice(0, 3), slice(L - 3, L)):
        p = torch.arange(L, device=dev)[sl]
        check(y[:, sl], turn(x[:, sl], cos, sin, p, True, 64), "bf16")


@pytest.mark.gpu
def test_rotary_more_work_than_one_launch_holds(dev):
    """2^33 channels copied one at a time, 2^32 threads: one row of heads, repeated by a stride of 0."""
    B, H, D, rot = (1 << 14) + 1, 4, (1 << 17) - 1, 6
    cos, sin = (torch.full((1, rot // 2), v, device=dev) for v in (0.6, 0.8))
    x = torch.randn(1, 1, H, D, device=dev).to(torch.bfloat16).expand(B, 1, H, D)
    y = rotary.apply_rotary(x, cos, sin, start=3)
    assert y.numel() > 1 << 33
    check(y[:1], turn(x[:1], cos, sin, torch.zeros(1, dtype=torch.int64, device=dev), True, 3), "bf16")
    for b in range(0, B, 1024):
        assert torch.equal(y[b:b + 1024], y[:1].expand(min(1024, B - b), 1, H, D))


@pytest.mark.gpu
def test_rotary_undoes_itself_and_keeps_lengths(dev):
    cos, sin = rotary.rotary_tables(128, 5000, device=dev)
    x = torch.randn(2, 300, 4, 128, device=dev, requires_grad=True)
    p = torch.arange(300, device=dev) + 4700
    y = rotary.apply_rotary(x, cos, sin, positions=p)
    (back,) = torch.autograd.grad(y, [x], y.detach())
    # cos^2 + sin^2 is 1 to 2 u each way; two turns of 3 u of the pair's sum
    assert (back - x).abs().max() <= 16 * U * x.abs().max()


@pytest.mark.gpu
def test_rotary_stream_graph_and_compile(dev):
    case = CASES[4]
    q, k, gq, gk, cos, sin, p = inputs(case, dev)

    def step(q, k):
        o = rotary.apply_rotary(q, cos, sin, k=k, positions=p, interleaved=False, start=128)
        return (*o, *torch.autograd.grad(o, [q, k], [gq, gk]))

    def leaves(a, b):
        return a.clone().requires_grad_(True), b.clone().requires_grad_(True)

    want = [t.detach().clone() for t in step(*leaves(q, k))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lv = leaves(q, k)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*lv)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    sq, sk = leaves(torch.zeros_like(q), torch.zeros_like(k))
    with torch.cuda.graph(graph):
        out = step(sq, sk)
    for r in range(3):
        with torch.no_grad():
            sq.copy_(q.roll(r, 0))
            sk.copy_(k.roll(r, 0))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*leaves(q.roll(r, 0), k.roll(r, 0)))
        assert all(torch.equal(a, b) for a, b in zip(want, out)), r

    def loss(q, k):
        a, b = rotary.apply_rotary(q, cos, sin, k=k, positions=p, interleaved=False, start=128)
        return (a * gq).sum() + (b * gk).sum()

    grads = []
    for f in (loss, torch.compile(loss, backend="aot_eager", fullgraph=True)):
        lq, lk = leaves(q, k)
        grads.append(torch.autograd.grad(f(lq, lk), [lq, lk]))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    torch.library.opcheck(torch.ops.cinnamon_amd.rotary, (q, k, cos, sin, p, False, 128, False))
    torch.library.opcheck(torch.ops.cinnamon_amd.rotary, (q, None, cos, sin, None, True, 0, True))


@pytest.mark.gpu
def test_rotary_feeds_the_indexer(dev):
    """Queries and keys of the indexer, turned in one call in front of its scores."""
    from cinnamon_amd import kernels
    torch.manual_seed(4)
    B, L, H, d = 2, 70, 4, 128
    cos, sin = rotary.rotary_tables(64, L, device=dev)
    q = torch.randn(B, L, H, d, device=dev).to(torch.bfloat16)
    k = torch.randn(B, L, d, device=dev).to(torch.bfloat16)
    w = torch.randn(B, L, H, device=dev)
    a, b = rotary.apply_rotary(q, cos, sin, k=k, interleaved=False)
    got = kernels.indexer_scores_fp8(a, b, w, d ** -0.5)
    ra = turn(q, cos, sin, None, False, 0)[0].to(torch.bfloat16).to(dev)
    rb = turn(k.unsqueeze(2), cos, sin, None, False, 0)[0].squeeze(2).to(torch.bfloat16).to(dev)
    # a bf16 value next to a tie may round the other way on either side (3 u against 2^-8: one in
    # thousands), and moves its e4m3 code by at most one step, 2^-3 of it
    want = kernels.indexer_scores_fp8(ra, rb, w, d ** -0.5)
    assert (got - want).norm() <= 1e-2 * want.norm()


def test_tables_are_64_bit_angles_rounded_once():
    cos, sin = rotary.rotary_tables(64, 100000)
    assert cos.shape == sin.shape == (100000, 32) and cos.dtype == torch.float32
    for p in (0, 1, 77, 99999):
        for i in (0, 1, 13, 31):
            a = p * 10000.0 ** (-2 * i / 64)
            # 64-bit angles of 10^5 are 1e-11 off, far under fp32's half step
            assert abs(cos[p, i].item() - math.cos(a)) <= U + 1e-10
            assert abs(sin[p, i].item() - math.sin(a)) <= U + 1e-10


def test_tables_scaled_for_long_contexts():
    def freqs(*a, **k):
        cos, sin = rotary.rotary_tables(*a, **k)
        return torch.atan2(sin[1].double(), cos[1].double()), (cos[0, 0].item())

    plain, one = freqs(64, 8)
    assert one == 1.0
    lin, _ = freqs(64, 8, scaling="linear", factor=4.0)
    assert torch.allclose(lin * 4, plain, rtol=1e-6)
    ntk, _ = freqs(64, 8, scaling="ntk", factor=4.0)
    assert torch.allclose(ntk[0], plain[0], rtol=1e-6) and torch.allclose(ntk[-1] * 4, plain[-1], rtol=1e-6)
    yarn, m = freqs(64, 8, scaling="yarn", factor=4.0, original_length=4096)
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-6
    ratio = plain / yarn
    assert torch.allclose(ratio[0], torch.ones(1, dtype=torch.float64)) and abs(ratio[-1].item() - 4) < 1e-5
    assert (ratio[1:] >= ratio[:-1] - 1e-6).all()
    # the ramp's ends: an index turning more than 32 times in 4096 positions stays, one turning less than once is divided
    turns = 4096 * plain / (2 * math.pi)
    assert (ratio[turns > 33 * 1.4] - 1).abs().max() < 1e-5 and (ratio[turns < 1 / 1.4] - 4).abs().max() < 1e-5
    _, m = freqs(64, 8, scaling="yarn", factor=4.0, original_length=4096, attention_factor=1.0)
    assert m == 1.0


def test_table_refusals():
    for bad in [dict(rot=3, length=4), dict(rot=0, length=4), dict(rot=4, length=-1), dict(rot=4, length=4, scaling="x"),
                dict(rot=2, length=4, scaling="ntk", factor=2.0), dict(rot=4, length=4, factor=0.5),
                dict(rot=4, length=4, base=1.0), dict(rot=4, length=4, scaling="yarn", factor=2.0, original_length=0),
                dict(rot=4, length=4, scaling="yarn", factor=2.0, beta_fast=1.0, beta_slow=2.0)]:
        with pytest.raises(AssertionError):
            rotary.rotary_tables(**bad)


def test_rotary_refusals():
    with FakeTensorMode():
        def fake(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        q, c = fake(2, 5, 3, 64), fake(10, 16)
        ap = rotary.apply_rotary
        for bad in [
            lambda: ap(torch.empty(2, 5, 3, 64), c, c),
            lambda: ap(fake(5, 64), c, c),
            lambda: ap(fake(2, 5, 3, 64, dtype=torch.float64), c, c),
            lambda: ap(q, c, c, k=fake(2, 5, 3, 64, dtype=torch.bfloat16)),
            lambda: ap(q, c, c, k=fake(2, 4, 3, 64)),
            lambda: ap(q, c, c, k=fake(2, 5, 3, 32)),
            lambda: ap(q, fake(10, 33), fake(10, 33)),
            lambda: ap(q, c, c, start=33),
            lambda: ap(q, c, c, start=-1),
            lambda: ap(q, c, fake(10, 15)),
            lambda: ap(q, c.bfloat16(), c.bfloat16()),
            lambda: ap(q, fake(4, 16), fake(4, 16)),
            lambda: ap(q, fake(10, 0), fake(10, 0)),
            lambda: ap(q, torch.empty(10, 16), torch.empty(10, 16)),
            lambda: ap(q, c.requires_grad_(True), c),
            lambda: ap(q, fake(10, 16), fake(10, 16), positions=fake(5)),
            lambda: ap(q, fake(10, 16), fake(10, 16), positions=fake(2, 5, dtype=torch.bool)),
            lambda: ap(q, fake(10, 16), fake(10, 16), positions=fake(4, dtype=torch.int64)),
            lambda: ap(q, fake(10, 16), fake(10, 16), positions=torch.empty(5, dtype=torch.int64)),
        ]:
            with pytest.raises(AssertionError):
                bad()
        a, b = ap(q, fake(10, 16), fake(10, 16), k=fake(2, 5, 64))
        assert a.shape == (2, 5, 3, 64) and b.shape == (2, 5, 64)


_OK = [1, 4, 4, 4, 1, 4, 4, 4, 1, None, 0, 0, 0, None, 0, 0, 0, 0, 0, 1, 1, 64, 1, 1, 8, 16, 32, 0, None, 0, 0, 1, 0, None]


@pytest.mark.parametrize("at,value", [(18, 5), (21, 16), (27, 33), (27, -1), (26, 31), (26, 0), (25, 15), (20, 9), (0, None),
                                      (4, None), (22, None), (19, -1), (17, 1)])
def test_rotary_c_refusals(at, value):
    args = list(_OK)
    args[at] = value
    with pytest.raises(ValueError):
        _lib.call("cin_rotary", *args)
