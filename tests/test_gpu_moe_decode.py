"""moe.moe_decode against its definition in 64 bits (GPU for the operator, CPU for the refusals).

With u = 2^-24: a product of K terms adds up along at most K of them in the matrix units' order and a few joins,
each rounding within u (the units do not round up to even everywhere: 2 u) of the running sum, itself within the sum of
magnitudes; random terms leave far less.  Bounds below: h within 8 sqrt(K) u of the magnitudes of its products, carried
through silu(a) b (slopes within 1.1 |b| and |silu(a)|), and h's parts keep 2^-16 of it (fp32 outputs: 2^-24); the
output sums those errors against |W3|, its own products' 8 sqrt(K) u, and one rounding.  Below the least normal number
nothing is kept: fp32 products and bf16 parts there have a spacing of up to 2^-133 and may count as zero, so each h
is off by 2^-126 more.
"""
import math
import threading

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, kernels, layers, moe

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E4M3 = torch.float8_e4m3fn


def values(w, s):
    """Weights in 64 bits."""
    if s is None:
        return w.double()
    R, C = w.shape[-2:]
    return w.float().double() * s.double().repeat_interleave(128, -2)[..., :R, :].repeat_interleave(128, -1)[..., :C]


def route(z, k, bias, score, groups, top_groups, group_top, renormalize, scale):
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, -1)
    choice = s if bias is None else s + bias.double()
    if groups > 1:
        per = choice.view(z.shape[0], groups, -1)
        best = per.sort(dim=-1, descending=True).values[..., :group_top].sum(-1)
        out = best.sort(dim=-1, descending=True, stable=True).indices[:, top_groups:]
        choice = per.clone().scatter_(1, out[..., None].expand(-1, -1, per.shape[2]), -math.inf).view_as(choice)
    idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, idx)
    if renormalize:
        w = w / (w.sum(-1, keepdim=True) + 1e-9)
    return idx, w * scale


def swiglu(x, w12, s12, w3, s3, weight, exact_h):
    """(the expert's output times weight, a bound of the kernel's error before its last rounding)"""
    W12, W3 = values(w12, s12), values(w3, s3)
    D, H = x.shape[1], W3.shape[1]
    a, b = (x @ W12.t()).chunk(2, -1)
    ma, mb = (x.abs() @ W12.abs().t()).chunk(2, -1)
    h = a * torch.sigmoid(a) * b * weight
    ea, eb = 8 * math.sqrt(D) * U * ma, 8 * math.sqrt(D) * U * mb
    eh = weight.abs() * (1.1 * ea * (b.abs() + eb) + eb * (a * torch.sigmoid(a)).abs()) + (8 * U + exact_h) * h.abs() + 2.0 ** -126
    return h @ W3.t(), (eh + 8 * math.sqrt(H) * U * h.abs()) @ W3.abs().t()


def definition(x, router, experts, k, bias=None, score="sigmoid", n_groups=1, top_groups=None, group_top=2, renormalize=True,
               scale=1.0, shared=None):
    xd = x.double()
    z = (xd[:, None, :] * router.double()).sum(-1)
    idx, w = route(z, k, bias, score, n_groups, top_groups or n_groups, group_top, renormalize, scale)
    out, err = torch.zeros_like(xd), torch.zeros_like(xd)
    part = 2.0 ** -24 if x.dtype == torch.float32 else 2.0 ** -16
    for e in idx.unique().tolist():
        t, j = (idx == e).nonzero(as_tuple=True)
        o, m = swiglu(xd[t], *(None if v is None else v[e] for v in experts), w[t, j][:, None], part)
        out[t] += o
        err[t] += m
    if shared is not None:
        o, m = swiglu(xd, *shared, torch.ones_like(xd[:, :1]), part)
        out, err = out + o, err + m
    return out, err, idx, w


def check(got, want):
    out, err, idx, w = want
    g, gi, gw = got
    assert g.shape == out.shape and gi.dtype == torch.int64 and gw.dtype == torch.float32
    assert torch.equal(gi, idx)
    assert ((gw.double() - w).abs() <= 2 * U * w.abs()).all()
    step = STEP[g.dtype]
    # (a sum over k experts rounds k times more)
    tol = step * out.abs() + (1 + step) * err * 1.1 + 2.0 ** -24 * (g.dtype == torch.float16)
    bad = ~((g.double() - out).abs() <= tol)
    assert not bad.any(), ((g.double() - out).abs() / tol)[bad].max()


def quantized(w):
    """Codes and scales of w [.., R, C] by 128 x 128 blocks."""
    R, C = w.shape[-2:]
    full = w.new_zeros(*w.shape[:-2], -(-R // 128) * 128, -(-C // 128) * 128)
    full[..., :R, :C] = w
    t = full.unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))
    s = t.abs().amax((-1, -3)).clamp_min(1e-4) / 448
    q = (t / s[..., None, :, None]).flatten(-2).flatten(-3, -2)[..., :R, :C].contiguous().to(E4M3)
    return q, s.contiguous()


def expert_weights(g, lead, D, H, wt):
    w12 = torch.randn(*lead, 2 * H, D, generator=g) * (1.5 / math.sqrt(D))
    w3 = torch.randn(*lead, D, H, generator=g) * (1.5 / math.sqrt(H))
    if wt == "bf16":
        return w12.bfloat16(), None, w3.bfloat16(), None
    return (*quantized(w12), *quantized(w3))


def to(dev, weights):
    return None if weights is None else tuple(None if t is None else t.to(dev) for t in weights)


def inputs(dev, T, D, H, E, dt, wt, Hs=0, router="fp32", seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, D, generator=g).to(DT[dt])
    r = (torch.randn(E, D, generator=g) * (1.5 / math.sqrt(D))).to(DT[router])
    return (x.to(dev), r.to(dev), to(dev, expert_weights(g, (E,), D, H, wt)),
            to(dev, expert_weights(g, (), D, Hs, wt)) if Hs else None)


CASES = [
    # T, D, H, E, k, x, weights, shared H, options
    (1, 16, 16, 1, 1, "fp32", "bf16", 0, {}),
    (1, 1024, 1024, 16, 2, "bf16", "fp8", 4096, {}),
    (3, 256, 128, 8, 8, "fp16", "fp8", 128, {"score": "softmax"}),
    (16, 528, 208, 20, 3, "fp32", "fp8", 80, {"renormalize": False, "scale": 2.5}),
    (17, 144, 400, 33, 4, "bf16", "bf16", 0, {"score": "softmax", "scale": 0.5}),
    (33, 272, 144, 6, 2, "fp32", "bf16", 48, {}),
    (64, 512, 256, 32, 8, "bf16", "fp8", 256, {"n_groups": 8, "top_groups": 4}),
    (65, 400, 112, 4, 4, "fp16", "bf16", 16, {"n_groups": 2, "top_groups": 2, "group_top": 1}),
    (100, 128, 384, 3, 2, "bf16", "fp8", 0, {}),
    (128, 1040, 272, 5, 5, "fp32", "fp8", 144, {"score": "softmax"}),
    (128, 96, 64, 1024, 16, "bf16", "fp8", 32, {"n_groups": 64, "top_groups": 7}),
    (40, 2000, 720, 60, 4, "bf16", "bf16", 0, {}),
    (128, 256, 128, 2, 1, "fp16", "fp8", 128, {}),
    # the shared expert's first product beside the gate in several units, and among the others where it is large
    (19, 1040, 272, 5, 2, "fp32", "bf16", 144, {}),
    (37, 784, 128, 12, 3, "bf16", "bf16", 208, {}),
    (29, 2048, 160, 6, 2, "fp16", "fp8", 1040, {}),
    (49, 1152, 128, 700, 2, "bf16", "fp8", 128, {}),
    (20, 512, 128, 4, 2, "bf16", "fp8", 8208, {}),
    (2, 256, 128, 4, 2, "fp16", "bf16", 8256, {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("router", ["fp32", "bf16"])
def test_against_the_definition(dev, case, router):
    T, D, H, E, k, dt, wt, Hs, options = case
    x, r, experts, shared = inputs(dev, T, D, H, E, dt, wt, Hs, router)
    bias = (torch.randn(E, generator=torch.Generator().manual_seed(2)) * 0.05).to(dev) if E > 4 else None
    kw = dict(bias=bias, shared=shared, **options)
    got = moe.moe_decode(x, r, experts, k, return_routing=True, **kw)
    check(got, definition(x, r, experts, k, **kw))
    again = moe.moe_decode(x, r, experts, k, **kw)
    assert torch.equal(again, got[0])
    # a token's result does not depend on the others
    if T > 1:
        for t in (0, T - 1):
            one = moe.moe_decode(x[t:t + 1], r, experts, k, return_routing=True, **kw)
            assert torch.equal(one[1], got[1][t:t + 1])
            check(one, tuple(v[t:t + 1] for v in definition(x, r, experts, k, **kw)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20])
def test_the_frameworks_experts(dev, T):
    """layers.GroupedExperts, with and without its weight cache, equals its codes; and the layer agrees with the
    gate and the routed experts, whose FP8 activations are off by up to 2^-4 of a value."""
    torch.manual_seed(3)
    E, D, H, k = 8, 256, 128, 2
    experts = layers.GroupedExperts(E, D, H).to(dev)
    with torch.no_grad():
        experts.w12.normal_(std=0.1)
        experts.w3.normal_(std=0.1)
    x, r = torch.randn(T, D, device=dev).bfloat16(), torch.randn(E, D, device=dev) * 0.1
    (w12, _, s12), (w3, _, s3) = layers.quantize_expert_weights(experts.w12.detach(), experts.w3.detach())
    weights = (w12.view(E, 2 * H, D), s12.view(E, 2 * H // 128, -1), w3.view(E, D, H), s3.view(E, D // 128, -1))
    got = moe.moe_decode(x, r, weights, k, return_routing=True)
    check(got, definition(x, r, weights, k))
    assert torch.equal(moe.moe_decode(x, r, experts, k), got[0])
    kernels.set_weight_cache(experts)
    for _ in range(2):
        assert torch.equal(moe.moe_decode(x, r, experts, k), got[0])
    with torch.no_grad():
        experts.w12.mul_(0.5)
        assert not torch.equal(moe.moe_decode(x, r, experts, k), got[0])
        experts.w12.mul_(2.0)
    idx, w = moe.moe_gate(x.float() @ r.t(), k)
    assert torch.equal(idx, got[1])
    routed, _ = moe.routed_experts(experts, x, idx, w)
    diff = (routed.double() - got[0].double()).norm() / got[0].double().norm()
    # two products of operands rounded to half a step of e4m3 (2^-4, an error of 2^-4 / sqrt(3) where uniform)
    assert diff < 2 * 2.0 ** -4


@pytest.mark.gpu
def test_ties_infinities_and_nan(dev):
    x, r, experts, shared = inputs(dev, 6, 256, 128, 12, "bf16", "fp8", 128)
    r[7], r[3] = r[2], r[2]  # equal logits go to the lowest index
    x[1, 5] = math.nan
    x[3] = 0
    x[4, 9] = math.inf
    out, idx, w = moe.moe_decode(x, r, experts, 12, shared=shared, return_routing=True)
    for t in (0, 2, 5):
        at = [idx[t].tolist().index(e) for e in (2, 3, 7)]
        assert at[1] == at[0] + 1 and at[2] == at[1] + 1
    good = torch.tensor([0, 2, 3, 5], device=dev)
    ref = definition(x[good], r, experts, 12, shared=shared)
    check((out[good], idx[good], w[good]), ref)
    assert (out[3] == 0).all() and torch.equal(idx[3], torch.arange(12, device=dev))
    assert out[1].isnan().all() and torch.equal(idx[1], torch.arange(12, device=dev)) and w[1].isnan().all()
    assert not torch.isfinite(out[4]).any()
    # fp32 and fp16 values that their first part rounds to infinity or that need all parts
    for dt, big in (("fp32", 3.0e38), ("fp16", 60000.0)):
        y, r2, e2, _ = inputs(dev, 2, 64, 32, 2, dt, "bf16")
        y[0] = y[0] * 1e-20 if dt == "fp32" else y[0] * 2.0 ** -10
        y[1, 3] = big
        r2[:, 3] = 0
        for v in (e2[0],):
            v[:, :, 3] = 0
        got = moe.moe_decode(y, r2, e2, 1, return_routing=True)
        check(got, definition(y, r2, e2, 1))


@pytest.mark.gpu
def test_logits_next_to_each_other(dev):
    """Experts whose logits differ by less than 32 bits hold are chosen in the order of the exact sums."""
    D, E = 64, 6
    x, _, experts, _ = inputs(dev, 1, D, 32, E, "fp32", "bf16")
    x.fill_(1.0)
    r = torch.zeros(E, D, device=dev)
    r[:, 0], r[:, 1] = 1.0, 2.0 ** -30 * torch.tensor([1.0, 4.0, 2.0, 6.0, 5.0, 3.0], device=dev)
    _, idx, _ = moe.moe_decode(x, r, experts, 6, return_routing=True)
    assert idx[0].tolist() == [3, 4, 1, 5, 2, 0]


@pytest.mark.gpu
def test_all_tokens_of_one_expert_and_unused_ones(dev):
    """128 tokens of one expert of 40; weights of experts that none chooses are not read: NaN there is no matter."""
    x, r, experts, _ = inputs(dev, 128, 128, 64, 40, "bf16", "bf16")
    bias = torch.full((40,), -100.0, device=dev)
    bias[17] = 100.0
    for e in range(40):
        if e != 17:
            experts[0][e] = math.nan
            experts[2][e] = math.nan
    got = moe.moe_decode(x, r, experts, 1, bias=bias, return_routing=True)
    assert (got[1] == 17).all()
    check(got, definition(x, r, experts, 1, bias=bias))


@pytest.mark.gpu
def test_strides_and_large_offsets(dev):
    x, r, experts, shared = inputs(dev, 9, 144, 80, 7, "bf16", "fp8", 48)
    want = moe.moe_decode(x, r, experts, 3, shared=shared)
    wide = torch.zeros(9, 400, dtype=x.dtype, device=dev)
    wide[:, 1:145] = x
    assert torch.equal(moe.moe_decode(wide[:, 1:145], r, experts, 3, shared=shared), want)
    rt = r.t().contiguous().t()
    assert torch.equal(moe.moe_decode(x.t().contiguous().t(), rt, experts, 3, shared=shared), want)
    off = [torch.empty(t.numel() + 3, dtype=t.dtype, device=dev)[3:].view(t.shape) for t in experts]
    for a, b in zip(off, experts):
        a.view(torch.uint8).copy_(b.view(torch.uint8)) if a.dtype == E4M3 else a.copy_(b)
    assert torch.equal(moe.moe_decode(x, r, tuple(off), 3, shared=shared), want)
    # experts beyond 2^32 bytes of the first: 70 of 2 x 4096 x 8192 codes
    E, D, H = 70, 8192, 4096
    g = torch.Generator(device=dev).manual_seed(4)
    w12 = torch.randint(0, 120, (E, 2 * H, D), dtype=torch.uint8, device=dev, generator=g).view(E4M3)
    w3 = torch.randint(0, 120, (E, D, H), dtype=torch.uint8, device=dev, generator=g).view(E4M3)
    s12 = torch.rand(E, 2 * H // 128, D // 128, device=dev, generator=g) * 1e-4
    s3 = torch.rand(E, D // 128, H // 128, device=dev, generator=g) * 1e-4
    x = torch.randn(2, D, device=dev, generator=g).bfloat16()
    r = torch.randn(E, D, device=dev, generator=g) * 0.01
    bias = torch.zeros(E, device=dev)
    bias[69] = 10.0
    got = moe.moe_decode(x, r, (w12, s12, w3, s3), 2, bias=bias, return_routing=True)
    assert (got[1][:, 0] == 69).all()
    check(got, definition(x, r, (w12, s12, w3, s3), 2, bias=bias))


@pytest.mark.gpu
def test_streams_threads_and_graphs(dev):
    x, r, experts, shared = inputs(dev, 24, 512, 256, 16, "bf16", "fp8", 256)
    want = moe.moe_decode(x, r, experts, 4, shared=shared, return_routing=True)
    empty = moe.moe_decode(x[:0], r, experts, 4, shared=shared, return_routing=True)
    assert empty[0].shape == (0, 512) and empty[1].shape == empty[2].shape == (0, 4)
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                results[i] = moe.moe_decode(x, r, experts, 4, shared=shared, return_routing=True)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = moe.moe_decode(x, r, experts, 4, shared=shared, return_routing=True)
    for seed in range(3):
        x.copy_(torch.randn(24, 512, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, moe.moe_decode(x, r, experts, 4, shared=shared, return_routing=True)))


@pytest.mark.gpu
def test_compiled(dev):
    x, r, experts, shared = inputs(dev, 5, 144, 64, 6, "bf16", "fp8", 32)

    def f(x, r, *w):
        return moe.moe_decode(x, r, w[:4], 2, shared=w[4:], return_routing=True)

    want = f(x, r, *experts, *shared)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, r, *experts, *shared)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # (opcheck itself cannot compute with codes)
    x, r, experts, shared = inputs(dev, 5, 144, 64, 6, "bf16", "bf16", 32)
    torch.library.opcheck(torch.ops.cinnamon_amd.moe_decode.default, (x, r, None, *experts, *shared, 2, 0, 1, 1, 2, True, 1.0))


@pytest.mark.gpu
def test_no_gradient(dev):
    x, r, experts, _ = inputs(dev, 2, 64, 32, 4, "bf16", "bf16")
    with pytest.raises(RuntimeError):
        moe.moe_decode(x.requires_grad_(), r, experts, 2).sum().backward()


def test_shapes_and_refusals():
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(*shape, dtype=dtype, device=device)

        f = torch.float32
        x, r = t(4, 256), t(8, 256)
        e16 = (t(8, 96, 256), None, t(8, 256, 48), None)
        e8 = (t(8, 96, 256, dtype=E4M3), t(8, 1, 2, dtype=f), t(8, 256, 48, dtype=E4M3), t(8, 2, 1, dtype=f))
        one = (t(64, 256), None, t(256, 32), None)
        for experts in (e16, e8):
            out, idx, w = moe.moe_decode(x, r, experts, 2, return_routing=True)
            assert out.shape == (4, 256) and idx.shape == w.shape == (4, 2) and idx.dtype == torch.int64 and w.dtype == f
        assert moe.moe_decode(x, r, e16, 2, shared=one).shape == (4, 256)
        for args, kw in [((t(129, 256), r, e16, 2), {}), ((t(4, 256, device="cpu"), r, e16, 2), {}),
                         ((x.double(), r, e16, 2), {}), ((x, t(8, 255), e16, 2), {}), ((x, t(8, 256, device="cpu"), e16, 2), {}),
                         ((x, t(1025, 256), e16, 2), {}), ((x, r, e16, 9), {}), ((x, r, e16, 0), {}), ((x, r, e16[:3], 2), {}),
                         ((x, r, (t(7, 96, 256), None, t(7, 256, 48), None), 2), {}),
                         ((x, r, (t(8, 96, 256), None, t(8, 256, 32), None), 2), {}),
                         ((t(4, 250), t(8, 250), (t(8, 96, 250), None, t(8, 250, 48), None), 2), {}),
                         ((x, r, (t(8, 80, 256), None, t(8, 256, 40), None), 2), {}),
                         ((x, r, (e16[0], e8[1], e16[2], e8[3]), 2), {}), ((x, r, (e8[0], None, e8[2], None), 2), {}),
                         ((x, r, (e8[0], t(8, 2, 2, dtype=f), *e8[2:]), 2), {}),
                         ((x, r, (t(8, 96, 256, dtype=f), None, t(8, 256, 48, dtype=f), None), 2), {}),
                         ((x, r, e8, 2), {"shared": one}), ((x, r, e16, 2), {"shared": e16}),
                         ((x, r, e16, 2), {"bias": t(8)}), ((x, r, e16, 2), {"bias": t(7, dtype=f)}), ((x, r, e16, 2), {"score": "relu"}),
                         ((x, r, e16, 2), {"n_groups": 3}), ((x, r, e16, 5), {"n_groups": 2, "top_groups": 1}),
                         ((x, r, e16, 2), {"group_top": 3}), ((x, r, e16, 2), {"n_groups": 2, "top_groups": 3})]:
            with pytest.raises(AssertionError):
                moe.moe_decode(*args, **kw)
        for sizes in [(7, 256, 128), (8, 128, 128), (8, 256, 96)]:  # the experts, the width, blocks of two experts
            with pytest.raises(AssertionError):
                moe.moe_decode(x, r, layers.GroupedExperts(*sizes), 2)


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    big = 1 << 20

    def call(dtype=0, T=4, D=256, E=8, k=2, H=48, Hs=0, ldx=256, ldr=256, router_dtype=1, score=0, groups=1, top=1, group_top=2, fp8=1,
             w12=big, s12=big, w3=big, s3=big, sw=None, x=big, out=big, ws=(big, 1 << 40)):
        return lib.cin_moe_decode(x, dtype, ldx, T, D, big, router_dtype, ldr, E, None, k, score, groups, top, group_top, 1, 1.0, fp8,
                                  w12, s12, w3, s3, H, sw, sw, sw, sw, Hs, out, big, big, *ws, None)

    for kw in [dict(dtype=3), dict(T=129), dict(T=-1), dict(D=250), dict(D=0), dict(E=1025), dict(E=0), dict(k=17), dict(k=9), dict(H=40),
               dict(H=65552), dict(Hs=8), dict(Hs=16), dict(sw=big), dict(ldx=255), dict(ldr=255), dict(router_dtype=9), dict(score=2),
               dict(groups=3), dict(top=2), dict(groups=4, top=1, k=3), dict(group_top=0), dict(w12=None), dict(s12=None), dict(w3=big + 8),
               dict(x=None), dict(out=None), dict(ws=(None, 0)), dict(ws=(big, 100)), dict(ws=(big + 8, 1 << 40))]:
        assert call(**kw) == _lib.CIN_ERR_ARG, kw
        assert _lib.last_error()
    assert call(T=0) == 0
    assert lib.cin_moe_decode_workspace(0, 1, 250, 8, 2, 48, 0) == -1
