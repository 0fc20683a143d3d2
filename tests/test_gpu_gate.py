"""moe.moe_gate against its definition in 64 bits (GPU), and its refusals (CPU).

Tolerances, all from fp32 roundings u = 2^-24: a score takes an exponential (2 u), its argument
(2 u), a sum and a reciprocal (3 u), under 8 u; the sum of k <= 16 scores adds 16 u and its
division and scale 4 u: a weight is within 32 u = 2^-19.  A softmax's sum over E experts adds at
most (E / 64 + 6) u, once to the scores and once to the weights.
"""
import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, moe

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(logits, k, bias=None, score="sigmoid", n_groups=1, top_groups=None, group_top=2, renormalize=True,
              scale=1.0, gw=None, gs=None):
    z = logits.detach().double().cpu().numpy()
    T, E = z.shape
    rows = np.arange(T)[:, None]
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            s = 1 / (1 + np.exp(-z))
        else:
            e = np.exp(z - z.max(1, keepdims=True))
            s = e / e.sum(1, keepdims=True)
    choice = s + (0 if bias is None else bias.double().cpu().numpy())
    order = np.where(np.isnan(choice), np.inf, choice)  # tests with NaN hold no inf
    top_groups = n_groups if top_groups is None else top_groups
    if n_groups > 1:
        n = E // n_groups
        per = np.sort(order.reshape(T, n_groups, n), axis=2)
        best = per[:, :, -min(group_top, n):].sum(2)
        out = np.argsort(-best, axis=1, kind="stable")[:, top_groups:]
        left = np.zeros((T, n_groups), bool)
        left[rows, out] = True
        left = np.repeat(left, n, axis=1)
    else:
        left = np.zeros((T, E), bool)
    # experts left out rank below every other, -inf included
    idx = np.lexsort((np.broadcast_to(np.arange(E), (T, E)), -order, left), axis=1)[:, :k]
    at = s[rows, idx]
    total = at.sum(1, keepdims=True) + 1e-9
    w = scale * (at / total if renormalize else at)
    r = {"idx": idx, "w": w, "scores": s}
    if gw is not None or gs is not None:
        ds = np.zeros_like(s) if gs is None else gs.double().cpu().numpy().copy()
        mag = np.abs(ds).max(1, keepdims=True)
        if gw is not None:
            g = gw.double().cpu().numpy() * scale
            if renormalize:
                ds[rows, idx] += g / total - (g * at).sum(1, keepdims=True) / total ** 2
                mag = mag + 2 * np.abs(g).max(1, keepdims=True) / total
            else:
                ds[rows, idx] += g
                mag = mag + np.abs(g).max(1, keepdims=True)
        r["dz"] = ds * s * (1 - s) if score == "sigmoid" else s * (ds - (s * ds).sum(1, keepdims=True))
        r["mag"] = mag * s
    return r


def check(got, ref, E, score, dlogits=None):
    more = 2 * (E / 64 + 6) * U if score == "softmax" else 0.0
    assert np.array_equal(got[0].cpu().numpy(), ref["idx"])
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.float32
    w = got[1].detach().double().cpu().numpy()
    np.testing.assert_allclose(w, ref["w"], rtol=32 * U + more, atol=1e-37)
    if len(got) == 3:
        np.testing.assert_allclose(got[2].detach().double().cpu().numpy(), ref["scores"], rtol=8 * U + more, atol=1e-37)
    if dlogits is not None:
        # fp32 errors of the terms (their magnitude times a weight's bound, twice: in a term and in the
        # sum taken from it), and the output's own rounding
        out = {torch.float32: U, torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}[dlogits.dtype]
        least = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}[dlogits.dtype]
        tol = 2 * out * np.abs(ref["dz"]) + (64 * U + 2 * more) * ref["mag"] + least
        d = np.abs(dlogits.double().cpu().numpy() - ref["dz"])
        assert (d <= tol).all(), (d / tol).max()


def make(T, E, dt, bias, seed, dev, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) * spread + torch.randn(E, generator=g) * 0.7).to(DT[dt]).to(dev)
    b = (torch.randn(E, generator=g) * 0.05).to(dev) if bias else None
    return logits, b, g


CASES = [
    # T, E, k, groups, top_groups, group_top, score, bias, renormalize, scale, dtype
    (1, 1, 1, 1, 1, 2, "sigmoid", False, True, 1.0, "fp32"),
    (1, 32, 8, 1, 1, 2, "sigmoid", True, True, 1.0, "fp32"),
    (5, 8, 8, 1, 1, 2, "softmax", False, True, 1.0, "bf16"),
    (1000, 16, 2, 1, 1, 2, "sigmoid", True, True, 1.0, "fp32"),
    (777, 16, 2, 1, 1, 2, "sigmoid", False, False, 2.5, "bf16"),
    (513, 33, 6, 1, 1, 2, "softmax", True, True, 1.0, "fp16"),
    (301, 64, 4, 8, 3, 2, "sigmoid", True, True, 1.0, "bf16"),
    (2049, 256, 8, 8, 4, 2, "sigmoid", True, True, 2.5, "bf16"),
    (130, 256, 8, 8, 4, 1, "softmax", False, False, 16.0, "fp32"),
    (499, 160, 6, 8, 3, 1, "softmax", False, True, 1.0, "fp16"),
    (67, 160, 6, 20, 2, 2, "softmax", True, True, 1.0, "bf16"),
    (19, 60, 5, 60, 7, 2, "sigmoid", True, True, 1.0, "fp32"),
    (19, 64, 16, 64, 16, 1, "sigmoid", True, True, 1.0, "fp32"),
    (33, 384, 16, 2, 1, 2, "sigmoid", True, True, 1.0, "bf16"),
    (9, 1000, 10, 4, 2, 2, "softmax", True, True, 1.0, "fp32"),
    (3, 4096, 16, 64, 8, 2, "sigmoid", True, True, 1.0, "bf16"),
    (3, 3001, 16, 1, 1, 2, "softmax", False, True, 1.0, "fp32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_gate_forward_and_backward(dev, case):
    T, E, k, G, tg, gt, score, bias, renorm, scale, dt = case
    logits, b, g = make(T, E, dt, bias, 3, dev)
    gw = torch.randn(T, k, generator=g).to(dev)
    gs = (torch.randn(T, E, generator=g) * 0.1).to(dev)
    kw = dict(bias=b, score=score, n_groups=G, top_groups=tg, group_top=gt, renormalize=renorm, scale=scale)
    ref = reference(logits, k, gw=gw, gs=gs, **kw)
    plain = moe.moe_gate(logits, k, **kw)
    assert len(plain) == 2
    check(plain, ref, E, score)
    leaf = logits.clone().requires_grad_(True)
    got = moe.moe_gate(leaf, k, return_scores=True, **kw)
    (dz,) = torch.autograd.grad([got[1], got[2]], [leaf], [gw, gs])
    assert dz.dtype == leaf.dtype
    check(got, ref, E, score, dz)
    # one of the two gradients alone
    ref_w = reference(logits, k, gw=gw, **kw)
    (dz,) = torch.autograd.grad(moe.moe_gate(leaf, k, **kw)[1], [leaf], gw)
    check(got, ref_w, E, score, dz)
    ref_s = reference(logits, k, gs=gs, **kw)
    (dz,) = torch.autograd.grad(moe.moe_gate(leaf, k, return_scores=True, **kw)[2], [leaf], gs)
    check(got, ref_s, E, score, dz)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,G,tg", [(16, 1, 1), (64, 8, 3), (256, 8, 4), (320, 4, 2), (2048, 1, 1)])
def test_gate_ties_take_the_lowest_index(dev, score, E, G, tg):
    g = torch.Generator().manual_seed(5)
    logits = torch.randint(-2, 3, (400, E), generator=g).to(torch.bfloat16).to(dev)
    for bias in (None, torch.zeros(E, device=dev), torch.randint(0, 2, (E,), generator=g).float().to(dev) * 0.25):
        kw = dict(bias=bias, score=score, n_groups=G, top_groups=tg)
        check(moe.moe_gate(logits, 8, **kw), reference(logits, 8, **kw), E, score)


@pytest.mark.gpu
@pytest.mark.parametrize("E,G,tg", [(32, 1, 1), (256, 8, 4), (512, 1, 1)])
def test_gate_orders_neighbours_that_fp32_cannot(dev, E, G, tg):
    """Saturated sigmoids and biases that differ in the last bits: the order is the 64-bit one."""
    g = torch.Generator().manual_seed(6)
    logits = (16 + torch.rand(300, E, generator=g) * 4).to(dev)      # 1 - s around 1e-8
    bias = (torch.randint(0, 3, (E,), generator=g).double() * 2.0 ** -23 + 0.5).float().to(dev)
    for b in (None, bias):
        kw = dict(bias=b, n_groups=G, top_groups=tg)
        check(moe.moe_gate(logits, 8, **kw), reference(logits, 8, **kw), E, "sigmoid")
    near = (torch.randn(300, 1, generator=g) + torch.randn(300, E, generator=g) * 1e-6).to(dev)
    for score in ("sigmoid", "softmax"):
        kw = dict(score=score, n_groups=G, top_groups=tg)
        check(moe.moe_gate(near, 8, **kw), reference(near, 8, **kw), E, score)


@pytest.mark.gpu
def test_gate_masked_experts_and_extreme_logits(dev):
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(64, 48, generator=g)
    logits[:, 5] = -float("inf")                          # an expert masked in the logits
    logits[1] = -float("inf")                             # a row whose mask leaves nothing
    logits[2, :40] = torch.finfo(torch.float32).min
    logits[3, 7] = 90.0
    logits[4] = -100.0
    logits = logits.to(dev)
    bias = torch.zeros(48)
    bias[11] = -float("inf")                              # and one masked in the bias
    for b in (None, bias.to(dev)):
        kw = dict(bias=b)
        got, ref = moe.moe_gate(logits, 6, **kw), reference(logits, 6, **kw)
        check(got, ref, 48, "sigmoid")
    rows = [r for r in range(64) if r != 1]               # (a softmax of nothing but -inf is NaN)
    kw = dict(score="softmax")
    check(moe.moe_gate(logits[rows], 6, **kw), reference(logits[rows], 6, **kw), 48, "softmax")
    one = torch.full((2, 48), -float("inf"), device=dev)
    idx, w = moe.moe_gate(one, 6, **kw)
    assert idx.tolist() == [list(range(6))] * 2 and torch.isnan(w).all()
    # with fewer finite choices than k, masked experts follow, the lowest first
    few = torch.zeros(1, 8, device=dev)
    masked = torch.tensor([-float("inf")] * 6 + [0.0, 0.0], device=dev)
    assert moe.moe_gate(few, 4, bias=masked)[0].tolist() == [[6, 7, 0, 1]]
    # every expert of the kept groups masked, those of the others not: the groups still decide
    assert moe.moe_gate(few, 2, bias=masked, n_groups=2, top_groups=1)[0].tolist() == [[6, 7]]


@pytest.mark.gpu
@pytest.mark.parametrize("E", [24, 200, 600])
def test_gate_nan_is_the_greatest_and_stays_in_its_row(dev, E):
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(10, E, generator=g).to(dev)
    logits[3, 17] = float("nan")
    idx, w = moe.moe_gate(logits, 4)
    assert idx[3, 0].item() == 17 and torch.isnan(w[3]).all()
    idx, w = moe.moe_gate(logits, 4, renormalize=False)
    assert torch.isnan(w[3, 0]) and torch.isfinite(w[3, 1:]).all()
    idx2, w2 = moe.moe_gate(logits, 4, n_groups=4, top_groups=2)
    assert idx2[3, 0].item() == 17
    good = [r for r in range(10) if r != 3]
    assert torch.isfinite(w[good]).all() and torch.isfinite(w2[good]).all()


@pytest.mark.gpu
def test_gate_strides_and_no_tokens(dev):
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(100, 70, generator=g).to(torch.bfloat16).to(dev)
    bias = torch.randn(140, generator=g).to(dev)[::2][:64]
    gw = torch.randn(4, 100, generator=g).to(dev).t()
    for view in (wide[:, 3:67], wide[::3, :64], wide[:64, :].t()[:64], wide[:1, :64].expand(100, 64)):
        kw = dict(bias=bias)
        leaf = view.detach().requires_grad_(True)
        got = moe.moe_gate(leaf, 4, **kw)
        ref = reference(view, 4, gw=gw[:view.shape[0]], **kw)
        (dz,) = torch.autograd.grad(got[1], [leaf], gw[:view.shape[0]])
        check(got, ref, 64, "sigmoid", dz)
    leaf = torch.empty(0, 64, device=dev, requires_grad=True)
    idx, w, s = moe.moe_gate(leaf, 4, return_scores=True)
    assert idx.shape == (0, 4) and w.shape == (0, 4) and s.shape == (0, 64)
    (dz,) = torch.autograd.grad(w.sum() + s.sum(), [leaf])
    assert dz.shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_gate_gradient_against_differences(dev, score):
    g = torch.Generator().manual_seed(10)
    logits = torch.randn(6, 20, generator=g).to(dev)
    gw, gs = torch.randn(6, 5, generator=g).to(dev), torch.randn(6, 20, generator=g).to(dev)
    leaf = logits.clone().requires_grad_(True)
    _, w, s = moe.moe_gate(leaf, 5, score=score, scale=1.5, return_scores=True)
    (dz,) = torch.autograd.grad([w, s], [leaf], [gw, gs])

    def value(z):
        r = reference(z, 5, score=score, scale=1.5)
        return (r["w"] * gw.double().cpu().numpy()).sum() + (r["scores"] * gs.double().cpu().numpy()).sum()

    h = 1e-5  # the difference's own error is about h^2, 1e-10, and 1e-16 / h = 1e-11
    for t in range(6):
        for e in range(0, 20, 3):
            z0, z1 = logits.double(), logits.double()
            z0[t, e] -= h
            z1[t, e] += h
            d = (value(z1) - value(z0)) / (2 * h)
            assert abs(d - dz[t, e].item()) < 1e-5


@pytest.mark.gpu
def test_gate_stream_graph_and_repeat(dev):
    logits, b, g = make(1500, 256, "bf16", True, 11, dev)
    gw = torch.randn(1500, 8, generator=g).to(dev)
    kw = dict(bias=b, n_groups=8, top_groups=4)

    def step(z):
        r = moe.moe_gate(z, 8, return_scores=True, **kw)
        return (*r, torch.autograd.grad(r[1], [z], gw)[0])

    want = [t.detach().clone() for t in step(logits.clone().requires_grad_(True))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaf = logits.clone().requires_grad_(True)
    with torch.cuda.stream(side):
        got = step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(logits).requires_grad_(True)
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in (0, 1, 2):
        z = logits.roll(seed, 0)
        with torch.no_grad():
            static.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        want = step(z.clone().requires_grad_(True))
        assert all(torch.equal(a, c) for a, c in zip(want, out)), seed


@pytest.mark.gpu
def test_gate_compiles(dev):
    logits, b, g = make(100, 64, "fp32", True, 12, dev)
    gw = torch.randn(100, 4, generator=g).to(dev)

    def step(z):
        i, w, s = moe.moe_gate(z, 4, bias=b, return_scores=True)
        return i, (w * gw).sum() + s.sum()

    grads = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaf = logits.clone().requires_grad_(True)
        i, loss = f(leaf)
        grads.append((i, torch.autograd.grad(loss, [leaf])[0]))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])
    torch.library.opcheck(torch.ops.cinnamon_amd.moe_gate, (logits, b, 4, 0, 1, 1, 2, True, 1.0, True))


@pytest.mark.gpu
def test_gate_feeds_the_routed_experts(dev):
    """A router's step as it is used: gate, routed experts, gradients down to the logits."""
    from cinnamon_amd import layers
    torch.manual_seed(13)
    T, D, E, k = 200, 256, 8, 2
    ex = layers.GroupedExperts(E, D, 256).to(dev)
    with torch.no_grad():
        ex.w12.normal_(std=0.05)
        ex.w3.normal_(std=0.05)
    x = torch.randn(T, D, device=dev).to(torch.bfloat16)
    z = torch.randn(T, E, device=dev)
    dout = torch.randn(T, D, device=dev)
    leaf = z.clone().requires_grad_(True)
    idx, w = moe.moe_gate(leaf, k)
    out, counts = moe.routed_experts(ex, x, idx, w)
    (dz,) = torch.autograd.grad(out, [leaf], dout)
    leaf2 = z.clone().requires_grad_(True)
    s = torch.sigmoid(leaf2)
    _, idx2 = s.topk(k)
    at = s.gather(1, idx2)
    w2 = at / (at.sum(-1, keepdim=True) + 1e-9)
    assert torch.equal(idx, idx2)
    out2, counts2 = moe.routed_experts(ex, x, idx2, w2)
    (dz2,) = torch.autograd.grad(out2, [leaf2], dout)
    assert torch.equal(counts, counts2)
    # the weights differ by at most 2^-19 of themselves on each side
    assert (out - out2).norm() <= 2 * 2.0 ** -19 * out2.norm()
    assert (dz - dz2).norm() <= 4 * 2.0 ** -19 * dz2.norm() + 64 * U * dout.norm() * out2.norm()


@pytest.mark.gpu
def test_gate_a_tie_behind_a_near_neighbour(dev):
    """Three sigmoids in one step of the ranked keys: the two equal ones are the greater, the lower
    index is not."""
    logits = torch.zeros(3, 256)
    for t, at in enumerate(([0, 1, 2], [3, 40, 41], [15, 16, 255])):
        logits[t, at] = torch.tensor([12.125, 12.1875, 12.1875])
    logits = logits.to(torch.bfloat16).to(dev)
    for b in (None, torch.zeros(256, device=dev), torch.full((256,), 0.25, device=dev)):
        assert moe.moe_gate(logits, 2, bias=b)[0].tolist() == [[1, 2], [40, 41], [16, 255]]
        assert moe.moe_gate(logits, 1, bias=b)[0].tolist() == [[1], [40], [16]]


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,G,tg", [(64, 1, 1), (256, 1, 1), (256, 8, 4), (1024, 1, 1), (1024, 16, 5)])
@pytest.mark.parametrize("about,step", [(12.0, 0.0625), (0.0, 2.0 ** -21), (-9.0, 0.0625)])
def test_gate_equal_logits_among_near_ones(dev, score, E, G, tg, about, step):
    """Few adjacent values, so that true ties and neighbours within a step of the keys meet at the border of
    the top k.  (Groups count by one expert where sums of two of the finest steps are equal in 64 bits.)"""
    g = torch.Generator().manual_seed(14)
    logits = (about + step * torch.randint(0, 6, (2000, E), generator=g)).to(torch.bfloat16).to(dev)
    for bias in (None, torch.zeros(E, device=dev), torch.full((E,), 0.5, device=dev)):
        for k in (2, 8):
            kw = dict(bias=bias, score=score, n_groups=G, top_groups=tg, group_top=1)
            check(moe.moe_gate(logits, k, **kw), reference(logits, k, **kw), E, score)
    spread = (torch.randn(2000, E, generator=g) * 6).to(torch.bfloat16).to(dev)
    tiny = (torch.randn(2000, E, generator=g) * 1e-4).to(torch.bfloat16).to(dev)
    for z in (spread, tiny):
        for bias in (None, torch.zeros(E, device=dev)):
            kw = dict(bias=bias, score=score)
            check(moe.moe_gate(z, 8, **kw), reference(z, 8, **kw), E, score)


@pytest.mark.gpu
@pytest.mark.parametrize("E,G", [(16, 4), (64, 4), (64, 32), (256, 8), (1024, 8), (1024, 64)])
def test_gate_groups_that_64_bits_cannot_tell_apart(dev, E, G):
    """Groups whose best logits differ by less than their scores in 64 bits hold are equal, whichever of
    them are equal in the logits too: the lowest stay."""
    g = torch.Generator().manual_seed(15)
    n = E // G
    best = torch.randint(1, 5, (300, G), generator=g).float() * 1e-18
    first = torch.tensor([[1.0, 2, 2, 2], [1, 3, 2, 2], [4, 1, 2, 2], [2, 2, 1, 2]]) * 1e-18
    best[:4, :4] = first
    best[:4, 4:] = -0.5
    best[200:] = torch.where(torch.rand(100, G, generator=g) < 0.5, best[200:], -0.25)
    logits = torch.full((300, G, n), -1.0)
    logits[torch.arange(300)[:, None], torch.arange(G), torch.randint(0, n, (300, G), generator=g)] = best
    logits = logits.flatten(1).to(dev)
    for tg in (1, 2, 3):
        for k in (1, min(2, tg * n)):
            kw = dict(n_groups=G, top_groups=tg, group_top=1)
            check(moe.moe_gate(logits, k, **kw), reference(logits, k, **kw), E, "sigmoid")
    for t in range(2):
        assert moe.moe_gate(logits[t:t + 1], 2, n_groups=G, top_groups=2, group_top=1)[0].div(n, rounding_mode="floor").tolist() == [[0, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("E", [8, 48, 256, 1500])
def test_gate_gradient_of_saturated_sigmoids(dev, E):
    """s (1 - s) = t / (1 + t)^2, t = e^-|z|, to the last bits also where s is next to 1.  t is within
    4 u, 1 + t and its reciprocal within 4 u more, so the factor within 4 + 2 * 5 + 2 u of itself, twice
    that here; a term of the weights' gradient is a sum over k of (gw_j - gw_i) s_i with errors of 8 u in
    the scores, 8 in the total and its square, 2 k in the sums."""
    g = torch.Generator().manual_seed(16)
    z = (torch.rand(200, E, generator=g) * 60 - 30).to(dev)
    gs = torch.randn(200, E, generator=g).to(dev)
    zd = z.double()
    t = torch.exp(-zd.abs())
    factor = t / (1 + t) ** 2
    leaf = z.clone().requires_grad_(True)
    s = moe.moe_gate(leaf, 2, return_scores=True)[2]
    (dz,) = torch.autograd.grad(s, [leaf], gs)
    want = gs.double() * factor
    assert ((dz.double() - want).abs() <= 32 * U * want.abs() + 1e-37).all()
    for k in (1, 2, min(8, E)):
        gw = torch.randn(200, k, generator=g).to(dev)
        for renormalize, scale in ((True, 1.0), (True, 2.5), (False, 1.0)):
            idx, w = moe.moe_gate(leaf, k, renormalize=renormalize, scale=scale)
            (dz,) = torch.autograd.grad(w, [leaf], gw)
            at = (1 / (1 + torch.exp(-zd))).gather(1, idx)
            gd = gw.double() * scale
            ds, size = gd, gd.abs()
            if renormalize:
                total = at.sum(1, keepdim=True) + 1e-9
                apart = gd[:, :, None] - gd[:, None, :]
                ds = ((apart * at[:, None]).sum(2) + 1e-9 * gd) / total ** 2
                size = ((apart.abs() * at[:, None]).sum(2) + 1e-9 * gd.abs()) / total ** 2
            want = torch.zeros_like(zd).scatter(1, idx, ds * factor.gather(1, idx))
            tol = torch.zeros_like(zd).scatter(1, idx, 2 * (32 + 2 * k) * U * size * factor.gather(1, idx)) + 1e-37
            assert ((dz.double() - want).abs() <= tol).all(), (k, renormalize)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("E", [8, 48, 256, 1500])
def test_gate_gradient_of_saturated_softmaxes(dev, dt, E):
    """s_j (ds_j - sum_e ds_e s_e) = s_j sum_e (ds_j - ds_e) s_e, also where one s is next to 1.  With c the
    gradient of the largest score's ds, the terms are |ds_e - c| s_e and |ds_j - c|, each off by a score's
    bound (8 u and the sum's E / 64 + 6), the sum's and two roundings more; twice that here."""
    g = torch.Generator().manual_seed(17)
    z = torch.randn(200, E, generator=g)
    z[torch.arange(200), torch.randint(0, E, (200,), generator=g)] += torch.rand(200, generator=g) * 60
    z[7] = 0.0                                             # all equal
    z = z.to(DT[dt]).to(dev)
    gs = (torch.randn(200, E, generator=g) + 3).to(dev)
    leaf = z.clone().requires_grad_(True)
    s = moe.moe_gate(leaf, 2, score="softmax", return_scores=True)[2]
    (dz,) = torch.autograd.grad(s, [leaf], gs)
    p, d = torch.softmax(z.double(), 1), gs.double()
    top = p.argmax(1, keepdim=True)
    c = d.gather(1, top)
    v = ((d - c) * p).sum(1, keepdim=True)
    want = p * (d - c - v)
    # (with several largest scores c is one of theirs: the largest difference of them more)
    same = torch.where(p == p.gather(1, top), (d - c).abs(), 0).amax(1, keepdim=True)
    size = p * ((d - c).abs() + ((d - c).abs() * p).sum(1, keepdim=True) + 2 * same)
    tol = 2 * (2 * (8 + E / 64 + 6) + 8) * U * size + 1e-37 + {"fp32": 0, "bf16": 2.0 ** -8}[dt] * want.abs()
    assert ((dz.double() - want).abs() <= tol).all()


def _fake(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_gate_refusals():
    with FakeTensorMode():
        z, b = _fake(4, 64), _fake(64)
        for bad in [
            lambda: moe.moe_gate(torch.empty(4, 64), 2),
            lambda: moe.moe_gate(_fake(64), 2),
            lambda: moe.moe_gate(_fake(4, 64, dtype=torch.float64), 2),
            lambda: moe.moe_gate(_fake(4, 4097), 2),
            lambda: moe.moe_gate(_fake(4, 0), 1),
            lambda: moe.moe_gate(z, 0),
            lambda: moe.moe_gate(z, 17),
            lambda: moe.moe_gate(_fake(4, 8), 9),
            lambda: moe.moe_gate(z, 2, score="tanh"),
            lambda: moe.moe_gate(z, 2, n_groups=7),
            lambda: moe.moe_gate(z, 2, n_groups=0),
            lambda: moe.moe_gate(_fake(4, 128), 2, n_groups=128),
            lambda: moe.moe_gate(z, 2, n_groups=8, top_groups=9),
            lambda: moe.moe_gate(z, 2, n_groups=8, top_groups=0),
            lambda: moe.moe_gate(z, 9, n_groups=8, top_groups=1),
            lambda: moe.moe_gate(z, 2, n_groups=8, group_top=3),
            lambda: moe.moe_gate(z, 2, bias=_fake(63)),
            lambda: moe.moe_gate(z, 2, bias=_fake(64, dtype=torch.bfloat16)),
            lambda: moe.moe_gate(z, 2, bias=torch.empty(64)),
        ]:
            with pytest.raises(AssertionError):
                bad()
        i, w, s = moe.moe_gate(z, 2, bias=b, return_scores=True)
        assert i.shape == w.shape == (4, 2) and s.shape == (4, 64)
        assert i.dtype == torch.int64 and w.dtype == s.dtype == torch.float32


@pytest.mark.parametrize("name,args", [
    ("cin_moe_gate", (1, 7, 64, None, 4, 64, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),     # dtype
    ("cin_moe_gate", (1, 0, 64, None, 4, 5000, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),   # experts
    ("cin_moe_gate", (1, 0, 63, None, 4, 64, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),     # rows overlap
    ("cin_moe_gate", (1, 0, 64, None, 4, 64, 17, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),    # k
    ("cin_moe_gate", (1, 0, 64, None, 4, 64, 2, 2, 1, 1, 2, 1, 1.0, 1, 1, None, None)),     # score
    ("cin_moe_gate", (1, 0, 64, None, 4, 64, 2, 0, 7, 1, 2, 1, 1.0, 1, 1, None, None)),     # groups
    ("cin_moe_gate", (1, 0, 64, None, 4, 64, 9, 0, 8, 1, 2, 1, 1.0, 1, 1, None, None)),     # too few left
    ("cin_moe_gate", (None, 0, 64, None, 4, 64, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),  # null
    ("cin_moe_gate", (1, 0, 64, None, 4, 64, 2, 0, 1, 1, 2, 1, 1.0, None, 1, None, None)),  # null
    ("cin_moe_gate_backward", (1, 0, 64, 4, 64, 2, 0, 1, 1.0, None, 1, 1, 1, None)),        # null
    ("cin_moe_gate_backward", (1, 0, 64, -1, 64, 2, 0, 1, 1.0, 1, 1, 1, 1, None)),          # T
    ("cin_moe_gate", (1, 0, 64, None, 1 << 28, 64, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),     # 2^32 threads
    ("cin_moe_gate", (1, 0, 512, None, 1 << 26, 512, 2, 0, 1, 1, 2, 1, 1.0, 1, 1, None, None)),
])
def test_gate_c_refusals(name, args):
    with pytest.raises(ValueError):
        _lib.call(name, *args)
