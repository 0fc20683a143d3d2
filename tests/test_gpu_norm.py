"""norm.block_norm and norm.rms_norm against their definition in 64 bits (GPU for the operators, CPU for
the refusals).

Every value is a chain of fp32 products and one or two sums over a row, rounded once to its type.  With u =
2^-24, a sum of D products by threads of up to 16 channels, a wave and 16 waves adds up along at most 16 + 6 +
16 roundings, so a row's 1 / rms is within (38 / 2 + 4) u of what its squares give; a value passes through two such sums and
fewer than 20 products.  With K = 100 that is within K u times the sum of the magnitudes of its terms (for a gradient:
twice, as the row's mean of its products passes through the forward's sums too).  A sum over rows adds the rows of a
workgroup, 32 lines of partial sums and their join: (T / workgroups + workgroups / 32 + 32) u more.
"""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, norm

U = 2.0 ** -24
K = 100
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}
EPS = 1e-6
NAMES = ("y", "residual", "weight", "post_weight", "gate", "residual_scale")


def definition(s, value, eps, gn, gx):
    """Both outputs and all gradients in 64 bits, each with the sum of its terms' magnitudes."""
    f = {n: None if t is None else t.detach().double() for n, t in s.items()}
    y, r, w, pw, g, a = (f[n] for n in NAMES)
    a = value if a is None else a
    w = 1.0 if w is None else w
    j = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = y if pw is None else y * j * pw
    gu = u if g is None else g * u
    x = gu if r is None else a * r + gu
    mx = gu.abs() + (0 if r is None else (a * r).abs())
    i = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * i * w
    spread = 1 + mx.square().mean(-1, keepdim=True).sqrt() * i  # the sum's own error in units of its rms
    out = {"normed": (n, i * abs(w) * mx * spread), "new": (x, mx)}
    gn = torch.zeros_like(y) if gn is None else gn.double()
    gx = torch.zeros_like(y) if gx is None else gx.double()
    t = gn * w
    dx = gx + i * (t - x * (i * i * (t * x).mean(-1, keepdim=True)))
    mdx = (gx.abs() + i * (t.abs() + mx * (i * i * (t.abs() * mx).mean(-1, keepdim=True)))) * spread
    if r is not None:
        out["residual"] = (a * dx, (abs(a) * mdx if not torch.is_tensor(a) else a.abs() * mdx))
    du = dx if g is None else g * dx
    mdu = mdx if g is None else g.abs() * mdx
    if pw is None:
        out["y"] = (du, mdu)
    else:
        t2, m2 = du * pw, mdu * pw.abs()
        out["y"] = (j * (t2 - y * (j * j * (t2 * y).mean(-1, keepdim=True))),
                    j * (m2 + y.abs() * (j * j * (m2 * y.abs()).mean(-1, keepdim=True))))
        out["post_weight"] = ((du * y * j).flatten(0, -2).sum(0), (mdu * y.abs() * j).flatten(0, -2).sum(0))
    out["weight"] = ((gn * x * i).flatten(0, -2).sum(0), (gn.abs() * mx * i * spread).flatten(0, -2).sum(0))
    if g is not None:
        out["gate"] = tuple(v.sum_to_size(g.shape) for v in (dx * u, mdx * u.abs()))
    if torch.is_tensor(a):
        out["residual_scale"] = tuple(v.sum_to_size(a.shape) if a.ndim else v.sum() for v in (dx * r, mdx * r.abs()))
    return out


def check(got, want, rows=0):
    v, mag = want
    g = got.detach().double()
    assert g.shape == v.shape
    tol = STEP[got.dtype] * v.abs() + (K + rows) * U * 2 * mag * (1 + STEP[got.dtype]) + LEAST[got.dtype]
    bad = ~((g - v).abs() <= tol)
    assert not bad.any(), ((g - v).abs() / tol)[bad].max()


def inputs(dev, shape, dt, rt, wt, post, gate, scale, weight=True, seed=1):
    gen = torch.Generator().manual_seed(seed)
    D = shape[-1]

    def make(*s, std=1.0, mean=0.0, t=None):
        return (torch.randn(*s, generator=gen) * std + mean).to(DT[t or dt]).to(dev)

    s = {"y": make(*shape, std=0.5), "residual": None if rt is None else make(*shape, std=2.0, t=rt),
         "weight": make(D, std=0.2, mean=1.0, t=wt) if weight else None,
         "post_weight": make(D, std=0.2, mean=1.0, t=wt) if post else None,
         "gate": {"none": lambda: None, "channel": lambda: make(D, std=0.5, t=wt), "row": lambda: make(*shape[:-1], 1, std=0.5, t=wt),
                  "element": lambda: make(*shape, std=0.5)}[gate](),
         "residual_scale": {"one": lambda: None, "number": lambda: None, "value": lambda: make(1, std=0.1, mean=0.9, t=wt),
                            "scalar": lambda: make(1, std=0.1, mean=0.9, t=wt).view(()),
                            "channel": lambda: make(D, std=0.1, mean=0.9, t=wt)}[scale]()}
    gn, gx = make(*shape, std=1e-2), None if rt is None else make(*shape, std=1e-2, t=rt)
    return s, 0.75 if scale == "number" else 1.0, gn, gx


def call(s, value):
    if s["residual"] is None:
        return norm.rms_norm(s["y"], s["weight"], EPS), None
    kw = dict(s)
    if kw["residual_scale"] is None:
        kw["residual_scale"] = value
    return norm.block_norm(kw.pop("y"), kw.pop("residual"), eps=EPS, **kw)


CASES = [
    # shape, y, residual, vectors, post, gate, scale
    ((1, 1), "fp32", "fp32", "fp32", True, "channel", "value"),
    ((1, 7168), "bf16", "bf16", "fp32", False, "none", "one"),
    ((3, 5, 64), "bf16", "fp32", "bf16", True, "row", "number"),
    ((700, 1024), "bf16", "fp32", "fp32", False, "none", "one"),
    ((2049, 512), "fp16", "fp16", "fp16", True, "element", "channel"),
    ((37, 1111), "fp16", "fp16", "fp16", True, "element", "channel"),
    ((129, 1025), "bf16", "bf16", "fp32", True, "channel", "value"),
    ((65, 1023), "fp32", "fp32", "fp32", True, "row", "scalar"),
    ((18, 7), "bf16", "bf16", "bf16", False, "channel", "channel"),
    ((300, 4096), "bf16", "bf16", "fp32", True, "channel", "value"),
    ((33, 8192), "fp16", "fp32", "fp32", True, "channel", "channel"),
    ((11, 8200), "bf16", "bf16", "fp32", True, "channel", "channel"),
    ((5, 16384), "fp32", "fp32", "fp32", True, "element", "channel"),
    ((6, 16383), "bf16", "fp32", "fp16", False, "none", "number"),
    ((600, 2048), "fp32", None, "fp32", False, "none", "one"),
    ((4, 130, 1536), "bf16", None, "fp32", False, "none", "one"),
    ((3000, 768), "fp16", "fp32", "fp32", False, "none", "one"),
    # several rows a workgroup
    ((5001, 1000), "bf16", "fp32", "fp32", True, "channel", "value"),
    ((2700, 1111), "fp16", "fp16", "fp16", True, "element", "channel"),
    ((1300, 4096), "bf16", "bf16", "fp32", True, "channel", "value"),
    ((1100, 3001), "bf16", "fp32", "bf16", False, "row", "number"),
    ((600, 6000), "bf16", "bf16", "fp32", True, "row", "channel"),
    ((520, 12000), "bf16", "bf16", "fp32", True, "channel", "channel"),
    ((515, 9001), "fp32", "fp32", "fp32", True, "element", "value"),
    ((530, 16384), "fp16", "fp32", "fp32", False, "none", "one"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(dev, case):
    s, value, gn, gx = inputs(dev, *case)
    ref = definition(s, value, EPS, gn, gx)
    n, x = call(s, value)
    assert n.dtype == s["y"].dtype
    check(n, ref["normed"])
    if x is not None:
        assert x.dtype == s["residual"].dtype
        check(x, ref["new"])
    leaves = {k: t.clone().requires_grad_() for k, t in s.items() if t is not None}
    n2, x2 = call({**s, **leaves}, value)
    assert torch.equal(n2, n) and (x is None or torch.equal(x2, x))
    outs, gs = ([n2], [gn]) if x is None else ([n2, x2], [gn, gx])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs, retain_graph=True)))
    T = math.prod(case[0][:-1])
    for k, g in grads.items():
        assert g.dtype == s[k].dtype
        # (each workgroup takes T / workgroups rows, and there are 16 times the CUs at most)
        check(g, ref[k], 0 if k in ("y", "residual") else T / min(T, 256) + 4096 / 32 + 32 + case[0][-1])
    again = torch.autograd.grad(outs, list(leaves.values()), gs, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(again, grads.values()))
    # each gradient alone, and that of one output alone
    for k, leaf in leaves.items():
        (g,) = torch.autograd.grad(outs, [leaf], gs, retain_graph=True)
        assert torch.equal(g, grads[k])
    if x is not None:
        for out, g, kept in ((n2, gn, 0), (x2, gx, 1)):
            one = definition(s, value, EPS, *((gn, None) if kept == 0 else (None, gx)))
            (dy,) = torch.autograd.grad(out, [leaves["y"]], g, retain_graph=True)
            check(dy, one["y"])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [96, 1100])
def test_strides(dev, dt, D):
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(41, 3 * D + 3, generator=gen).to(DT[dt]).to(dev)
    y, r, gate = wide[:, 1:1 + D], wide[:, D + 2:2 * D + 2], wide[:, 2 * D + 3:]
    w = torch.randn(2 * D, generator=gen).to(dev)[::2]
    s = {"y": y, "residual": r, "weight": w, "post_weight": w, "gate": gate, "residual_scale": None}
    leaves = {k: t.detach().requires_grad_() for k, t in s.items() if t is not None}
    n, x = call({**s, **leaves}, 0.5)
    gn, gx = torch.randn(D, 41, generator=gen).to(DT[dt]).to(dev).t(), torch.ones(1, 1, dtype=DT[dt], device=dev).expand(41, D)
    ref = definition(s, 0.5, EPS, gn, gx)
    check(n, ref["normed"])
    check(x, ref["new"])
    for k, g in zip(leaves, torch.autograd.grad([n, x], list(leaves.values()), [gn, gx])):
        check(g, ref[k], 200)
    # columns of a transposed tensor, rows that repeat
    yt = torch.randn(D, 41, generator=gen).to(DT[dt]).to(dev).t()
    rt = r[:1].expand(41, D)
    n, x = norm.block_norm(yt, rt, w, eps=EPS)
    ref = definition({**s, "y": yt, "residual": rt, "post_weight": None, "gate": None}, 1.0, EPS, None, None)
    check(n, ref["normed"])
    check(x, ref["new"])


@pytest.mark.gpu
def test_gate_of_rows_with_a_stride(dev):
    gen = torch.Generator().manual_seed(4)
    y, r = (torch.randn(2, 9, 256, generator=gen).bfloat16().to(dev) for _ in range(2))
    gate = torch.randn(2, 9, 5, generator=gen).to(dev)[..., 3:4]
    for gt in (gate, gate[:, :1].expand(2, 9, 1)):
        s = {"y": y, "residual": r, "weight": None, "post_weight": None, "gate": gt, "residual_scale": None}
        n, x = call(s, 1.0)
        ref = definition(s, 1.0, EPS, None, None)
        check(n, ref["normed"])
        check(x, ref["new"])


@pytest.mark.gpu
def test_differences(dev):
    """The gradients against differences of the 64-bit definition along random directions."""
    s, value, gn, gx = inputs(dev, (6, 200), "fp32", "fp32", "fp32", True, "channel", "channel")
    leaves = {k: t.clone().requires_grad_() for k, t in s.items()}
    n, x = call(leaves, value)
    grads = dict(zip(leaves, torch.autograd.grad([n, x], list(leaves.values()), [gn, gx])))

    def total(t):
        out = definition(t, value, EPS, None, None)
        return ((out["normed"][0] * gn.double()).sum() + (out["new"][0] * gx.double()).sum()).item()

    gen = torch.Generator().manual_seed(5)
    for k in NAMES:
        d = torch.randn(s[k].shape, generator=gen, dtype=torch.float64).to(dev)
        h = 1e-5
        diff = (total({**s, k: s[k].double() + h * d}) - total({**s, k: s[k].double() - h * d})) / (2 * h)
        want = (grads[k].double() * d).sum().item()
        # (differences: h^2 and 1e-16 / h of the whole; gradients: fp32)
        assert abs(diff - want) <= 1e-5 * (grads[k].double() * d).abs().sum().item() + 1e-8


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 1536])
def test_rows_with_nothing_infinities_and_nan(dev, D):
    """Such a row keeps to itself; a row of zeros gives zeros."""
    gen = torch.Generator().manual_seed(6)
    y, r = (torch.randn(9, D, generator=gen).to(dev) for _ in range(2))
    w = torch.ones(D, device=dev)
    y[1], r[1] = 0, 0
    y[3, 5] = math.nan
    r[5, 7] = math.inf
    good = torch.tensor([0, 2, 4, 6, 7, 8], device=dev)
    leaf = y.clone().requires_grad_()
    n, x = norm.block_norm(leaf, r, w, post_weight=w)
    n1, x1 = norm.block_norm(y[good], r[good], w, post_weight=w)
    assert torch.equal(n[good], n1) and torch.equal(x[good], x1)
    assert (n[1] == 0).all() and (x[1] == 0).all()
    assert n[3].isnan().all() and x[3].isnan().all()
    assert n[5].isnan().sum() == 1 and (n[5][:7] == 0).all() and torch.isinf(x[5, 7])
    (dy,) = torch.autograd.grad([n, x], [leaf], [torch.ones_like(n), torch.ones_like(x)])
    other = y[good].clone().requires_grad_()
    n1, x1 = norm.block_norm(other, r[good], w, post_weight=w)
    (d1,) = torch.autograd.grad([n1, x1], [other], [torch.ones_like(n1), torch.ones_like(x1)])
    assert torch.equal(dy[good], d1) and dy[3].isnan().all() and torch.isfinite(dy[1]).all()


@pytest.mark.gpu
def test_no_rows(dev):
    s, value, gn, gx = inputs(dev, (0, 128), "bf16", "bf16", "fp32", True, "channel", "value")
    leaves = {k: t.clone().requires_grad_() for k, t in s.items()}
    n, x = call(leaves, value)
    assert n.shape == x.shape == (0, 128)
    grads = dict(zip(leaves, torch.autograd.grad([n, x], list(leaves.values()), [gn, gx])))
    assert all(g.shape == s[k].shape for k, g in grads.items())
    assert all((grads[k] == 0).all() for k in NAMES[2:])


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """Rows whose elements lie beyond 2^32 bytes and 2^31 elements of their tensor's start."""
    D, stride = 64, 1 << 27
    base = torch.zeros(18 * stride + D, dtype=torch.bfloat16, device=dev)
    y = torch.as_strided(base, (19, D), (stride, 1))
    gen = torch.Generator().manual_seed(7)
    y.copy_(torch.randn(19, D, generator=gen).bfloat16())
    n = norm.rms_norm(y, None, EPS)
    assert torch.equal(n, norm.rms_norm(y.contiguous(), None, EPS))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,scale", [((130, 1536), "value"), ((9, 8192), "channel"), ((70, 256), "channel")])
def test_another_stream_and_a_graph(dev, shape, scale):
    s, value, gn, gx = inputs(dev, shape, "bf16", "bf16", "fp32", True, "channel", scale)
    leaves = {k: t.clone().requires_grad_() for k, t in s.items()}
    n, x = call(leaves, value)
    eager = torch.autograd.grad([n, x], list(leaves.values()), [gn, gx], retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = {k: t.clone().requires_grad_() for k, t in s.items()}
        n2, x2 = call(held, value)
        on_side = torch.autograd.grad([n2, x2], list(held.values()), [gn, gx])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(eager, on_side))
    # (leaves that no eager graph holds any more: torch cannot capture a backward through such)
    held = {k: t.clone().requires_grad_() for k, t in s.items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n3, x3 = call(held, value)
        captured = torch.autograd.grad([n3, x3], list(held.values()), [gn, gx])
    for seed in range(3):
        fresh, _, _, _ = inputs(dev, shape, "bf16", "bf16", "fp32", True, "channel", scale, seed=seed)
        with torch.no_grad():
            for k in held:
                held[k].copy_(fresh[k])
        graph.replay()
        torch.cuda.synchronize()
        m, v = call({k: t.clone().requires_grad_() for k, t in fresh.items()}, value)
        assert torch.equal(n3, m) and torch.equal(x3, v)
        mine = {k: t.clone().requires_grad_() for k, t in fresh.items()}
        m, v = call(mine, value)
        want = torch.autograd.grad([m, v], list(mine.values()), [gn, gx])
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


@pytest.mark.gpu
def test_compiled(dev):
    s, value, gn, gx = inputs(dev, (33, 1100), "bf16", "fp32", "fp32", True, "row", "value")
    leaves = {k: t.clone().requires_grad_() for k, t in s.items()}

    def f(*t):
        d = dict(zip(leaves, t))
        n, x = norm.block_norm(d.pop("y"), d.pop("residual"), **d)
        return n * 2, x, norm.rms_norm(x)

    outs = f(*leaves.values())
    want = torch.autograd.grad(outs, list(leaves.values()), [gn, gx, gx])
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves.values())
    assert all(torch.equal(a, b) for a, b in zip(got, outs))
    grads = torch.autograd.grad(got, list(leaves.values()), [gn, gx, gx])
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.gpu
def test_operator_checks(dev):
    s, value, _, _ = inputs(dev, (5, 96), "bf16", "fp32", "fp32", True, "channel", "value")
    args = [s[k].clone().requires_grad_() for k in NAMES]
    torch.library.opcheck(torch.ops.cinnamon_amd.block_norm.default, (*args, value, EPS))
    torch.library.opcheck(torch.ops.cinnamon_amd.block_norm.default, (args[0], None, args[2], None, None, None, value, EPS))


def test_shapes_on_fake_tensors():
    with FakeTensorMode():
        y = torch.empty(2, 5, 96, dtype=torch.bfloat16, device="cuda")
        r, w, gate = (torch.empty(*s, device="cuda") for s in ((2, 5, 96), (96,), (2, 5, 1)))
        n, x = norm.block_norm(y, r, w, gate=gate)
        assert n.shape == y.shape and n.dtype == y.dtype and x.shape == r.shape and x.dtype == r.dtype
        grads = torch.ops.cinnamon_amd.block_norm_backward(n, x, y, r, w, None, gate, None, torch.empty(20, device="cuda"), 1.0,
                                                           [True, True, False, False, True, False])
        assert [g.shape for g in grads] == [y.shape, r.shape, (0,), (0,), gate.shape, (0,)]
        assert [g.dtype for g in grads[:2]] == [y.dtype, r.dtype]
        assert norm.rms_norm(y, w).shape == y.shape


def test_refusals():
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(*shape, dtype=dtype, device=device)

        y, r, w = t(4, 64), t(4, 64), t(64, dtype=torch.float32)
        for args, kw in [((t(4, 64, device="cpu"), r, w), {}), ((t(4, 64, dtype=torch.float64), r, w), {}),
                         ((y, t(4, 63), w), {}), ((y, None, w), {}), ((y, t(4, 64, dtype=torch.float16), w), {}),
                         ((t(4, 64, dtype=torch.float32), r, w), {}), ((y, r, t(63)), {}), ((y, r, t(4, 64)), {}),
                         ((y, r, w), {"post_weight": t(63)}), ((y, r, w), {"gate": t(4)}), ((y, r, w), {"gate": t(3, 1)}),
                         ((y, r, w), {"gate": t(4, 64, dtype=torch.float32)}), ((y, r, w), {"residual_scale": t(4)}),
                         ((y, r, w), {"residual_scale": t(64, device="cpu")}), ((y, r, t(64, dtype=torch.int32)), {}),
                         ((t(2, 16385), t(2, 16385)), {}), ((t(2, 0), t(2, 0)), {})]:
            with pytest.raises(AssertionError):
                norm.block_norm(*args, **kw)
        with pytest.raises(AssertionError):
            norm.rms_norm(y, t(4, 64))


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    y, r, w = (1 << 20, 0, 64), (1 << 20, 0, 64), (1 << 20, 1)
    sizes, none2, gate, scale = (4, 64), (None, 0), (None, 0, 0, 0), (None, 0, 0, 1.0)

    def forward(y=y, r=r, sizes=sizes, w=w, pw=none2, gate=gate, scale=scale, n=1 << 20):
        return lib.cin_block_norm(*y, *r, *sizes, *w, *pw, *gate, *scale, 1e-6, n, None, None, None)

    big = 1 << 20
    for kw in [dict(y=(big, 7, 64)), dict(y=(big, 0, 63)), dict(y=(None, 0, 64)), dict(r=(big, 2, 64)), dict(r=(big, 0, 63)),
               dict(sizes=(4, 0)), dict(sizes=(4, 16385)), dict(sizes=(-1, 64)), dict(w=(big, 5)), dict(pw=(big, 5)),
               dict(gate=(None, 0, 1, 0)), dict(gate=(big, 0, 0, 0)), dict(gate=(big, 0, 4, 64)), dict(gate=(big, 1, 3, 64)),
               dict(gate=(big, 0, 3, 63)), dict(gate=(big, 0, 2, 0)), dict(scale=(None, 0, 1, 1.0)),
               dict(scale=(big, 0, 0, 1.0)), dict(scale=(big, 9, 2, 1.0)), dict(n=None)]:
        assert forward(**kw) == _lib.CIN_ERR_ARG, kw
        assert _lib.last_error()
    assert forward(sizes=(0, 64)) == 0

    def backward(dw=big, dr=big, ws=(big, 1 << 30), stats=big, ldgn=64, r=r, dscale=None):
        return lib.cin_block_norm_backward(*y, *r, *sizes, *w, *none2, *gate, *scale, stats, big, ldgn, None, 0, big, dr, dw, None,
                                           None, dscale, *ws, None)

    for kw in [dict(ws=(None, 0)), dict(ws=(big, 100)), dict(stats=None), dict(ldgn=63), dict(r=(None, 0, 64)), dict(dscale=big)]:
        assert backward(**kw) == _lib.CIN_ERR_ARG, kw
    assert lib.cin_block_norm_workspace(5, 16385) == -1 and lib.cin_block_norm_workspace(-1, 64) == -1
    assert lib.cin_block_norm_workspace(0, 64) == 0
