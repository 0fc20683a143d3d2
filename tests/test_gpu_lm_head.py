"""lm_head.linear_cross_entropy against its definition in 64 bits (GPU), and its refusals (CPU).

Tolerances.  u = 2^-24, step = half a step of the type (bf16 2^-8, fp16 2^-11, fp32 u).
  logits     fp32 sums of D exact products: within D u S, S = sum_d |x_d w_d|, e = D u max S
  loss       2 e (maximum and target's logit), and 64 u for the exponentials, their sum and the log
  dz         its own rounding, step |dz|, and p (2 e + 16 u + 64 u); fp16 is scaled so that the
             largest row gradient tops 2^15: what lies under fp16's least number is off by 2^-39 of it
  dx, dw     the sum of dz's errors times |w| or |x|, K u sum |dz w| for K fp32 additions, and the
             output's rounding
These hold for each value in the worst case.  Roundings point both ways, so over a whole tensor the
norm of the error stays under that of one rounding to the type and of sqrt(K) fp32 ones: twice the
step (one for dz, one for the output), and 4 sqrt(K + D) u.
"""
import math

import pytest
import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, lm_head

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": U}
LEAST = {"bf16": 1e-37, "fp16": 2.0 ** -24, "fp32": 1e-37}


def reference(x, w, y, ignore=-100, reduction="mean", grad=None):
    """loss, dx, dw in 64 bits and the worst-case error of each value."""
    dt = {v: k for k, v in DT.items()}[x.dtype]
    x, w, y = x.detach().double(), w.detach().double(), y.reshape(-1).long()
    x = x.reshape(-1, x.shape[-1])
    (T, D), V = x.shape, w.shape[0]
    kept = y != ignore
    n = int(kept.sum())
    z = x @ w.t()
    e = D * U * (x.abs() @ w.abs().t()).amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = torch.where(kept, y, 0)[:, None]
    rows = torch.where(kept, (lse - z.gather(1, at))[:, 0], 0)
    rtol = torch.where(kept, 2 * e[:, 0] + 64 * U + 2 * U * rows, 0)
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n if n else torch.tensor(math.nan)}[reduction]
    ltol = {"none": rtol, "sum": rtol.sum(), "mean": rtol.sum() / max(n, 1)}[reduction]
    g = torch.ones(T, dtype=torch.float64, device=x.device) if grad is None else grad.double().reshape(-1).expand(T)
    g = torch.where(kept, g, 0) / (max(n, 1) if reduction == "mean" else 1)
    p = torch.exp(z - lse)
    dz = p.scatter_add(1, at, -torch.ones_like(at, dtype=torch.float64)) * g[:, None]
    dz_err = STEP[dt] * dz.abs() + p * g.abs()[:, None] * (2 * e + 80 * U) + 4 * U * dz.abs()
    if dt == "fp16":
        dz_err = dz_err + 2.0 ** -39 * g.abs().max()
    dz_err = torch.where(kept[:, None], dz_err, 0)
    dx, dw = dz @ w, dz.t() @ x
    dx_tol = dz_err @ w.abs() + V * U * (dz.abs() @ w.abs()) + STEP[dt] * dx.abs()
    dw_tol = dz_err.t() @ x.abs() + T * U * (dz.abs().t() @ x.abs()) + STEP[dt] * dw.abs()
    return (loss, ltol), (dx, dx_tol), (dw, dw_tol)


def near(got, ref, tol, dt, K):
    got = got.detach().double().reshape(ref.shape)
    assert torch.isfinite(got).all()
    d = (got - ref).abs()
    bound = 1.01 * tol + LEAST[dt]
    assert (d <= bound).all(), (d / bound).max().item()
    norm = 2 * STEP[dt] + 4 * math.sqrt(K) * U
    assert d.norm() <= norm * ref.norm() + LEAST[dt] * math.sqrt(d.numel()), (d.norm() / ref.norm()).item()


def make(T, V, D, dt, ignored, dev, seed=1, ignore=-100):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) * (2 / math.sqrt(D))
    y = torch.randint(0, V, (T,), generator=g)
    x = torch.randn(T, D, generator=g) + torch.rand(T, 1, generator=g) * 2 * w[y]
    y = torch.where(torch.rand(T, generator=g) < ignored, ignore, y)
    return x.to(DT[dt]).to(dev), w.to(DT[dt]).to(dev), y.to(dev), g


SHAPES = [
    # T, V, D, ignored
    (1, 1, 1, 0.0), (1, 1000, 64, 0.0), (2, 7, 130, 0.0), (16, 3201, 96, 0.0), (65, 64, 8, 0.3), (255, 257, 64, 0.0),
    (257, 513, 129, 0.5), (300, 2049, 192, 0.1), (513, 5003, 320, 0.4), (1000, 300, 777, 0.9), (130, 1024, 1024, 0.0),
    (3, 20011, 33, 0.0), (128, 3001, 256, 0.2), (129, 700, 2048, 0.0), (33, 5000, 65, 0.0), (20, 260, 4097, 0.1), (32, 9000, 512, 0.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_loss_and_gradients(dev, shape, dt):
    T, V, D, ignored = shape
    x, w, y, g = make(T, V, D, dt, ignored, dev)
    for reduction in ("mean", "sum", "none"):
        grad = torch.randn(T, generator=g).to(dev) if reduction == "none" else torch.randn((), generator=g).to(dev)
        if reduction == "mean" and int((y >= 0).sum()) == 0:
            y = y.clone()
            y[0] = 0
        (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w, y, reduction=reduction, grad=grad)
        with torch.no_grad():
            plain = lm_head.linear_cross_entropy(x, w, y, reduction=reduction)
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        got = lm_head.linear_cross_entropy(xl, wl, y, reduction=reduction)
        assert got.dtype == torch.float32 and got.shape == loss.shape and torch.equal(plain, got.detach())
        assert ((got.detach().double() - loss).abs() <= ltol).all()
        a, b = torch.autograd.grad(got, [xl, wl], grad)
        assert a.dtype == b.dtype == x.dtype and a.shape == x.shape and b.shape == w.shape
        near(a, dx, dxt, dt, V + D)
        near(b, dw, dwt, dt, T + D)
        assert (a[y == -100] == 0).all()
        if reduction == "sum":  # one gradient alone
            (a1,) = torch.autograd.grad(lm_head.linear_cross_entropy(xl, w, y, reduction=reduction), [xl], grad)
            (b1,) = torch.autograd.grad(lm_head.linear_cross_entropy(x, wl, y, reduction=reduction), [wl], grad)
            assert torch.equal(a1, a) and torch.equal(b1, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,D", [(3, (1 << 20) + 1000, 64), (9000, 70001, 64)])
def test_more_than_one_piece_of_the_vocabulary(dev, T, V, D, dt):
    if dt == "fp32" and T > 100:
        V = 35001
    x, w, y, g = make(T, V, D, dt, 0.1, dev)
    y[0] = V - 1
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w, y)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = lm_head.linear_cross_entropy(xl, wl, y)
    assert (got.detach().double() - loss).abs() <= ltol
    a, b = torch.autograd.grad(got, [xl, wl])
    near(a, dx, dxt, dt, V + D)
    near(b, dw, dwt, dt, T + D)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_ignored_and_impossible_targets(dev, dt):
    x, w, y, g = make(40, 300, 72, dt, 0.0, dev)

    def run(y, **kw):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = lm_head.linear_cross_entropy(xl, wl, y, **kw)
        return (loss.detach(), *torch.autograd.grad(loss.sum(), [xl, wl]))

    none = torch.full_like(y, -100)
    for reduction, want in (("sum", 0.0), ("mean", math.nan), ("none", 0.0)):
        loss, dx, dw = run(none, reduction=reduction)
        assert torch.isnan(loss).all() if math.isnan(want) else (loss == want).all()
        assert (dx == 0).all() and (dw == 0).all()
    # an ignore_index inside the vocabulary
    yi = torch.where(torch.arange(40, device=dev) % 3 == 0, 7, y)
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w, yi, ignore=7)
    got = run(yi, ignore_index=7)
    assert (got[0].double() - loss).abs() <= ltol
    near(got[1], dx, dxt, dt, 372)
    near(got[2], dw, dwt, dt, 112)
    # impossible targets: their rows only in the loss and in dx
    for bad in (300, -1, 2 ** 40, -(2 ** 40)):
        yb = y.clone()
        yb[5] = bad
        loss, dx, dw = run(yb, reduction="none")
        assert torch.isnan(loss[5]) and torch.isfinite(loss).sum() == 39
        assert torch.isnan(dx[5]).all() and torch.isfinite(dx).sum() == 39 * 72 and torch.isnan(dw).all()
        assert torch.isnan(run(yb)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_strides_shapes_and_targets_types(dev, dt):
    T, V, D = 60, 500, 128
    x, w, y, g = make(T, V, D, dt, 0.2, dev)
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w, y)
    wide = torch.zeros(T, D + 9, dtype=x.dtype, device=dev)
    wide[:, 5:5 + D] = x
    ww = torch.zeros(V, 2 * D + 8, dtype=x.dtype, device=dev)
    ww[:, :D] = w
    wo = torch.zeros(V * D + 1, dtype=x.dtype, device=dev)
    wo[1:] = w.reshape(-1)
    xs = [x, wide[:, 5:5 + D], x.t().contiguous().t(), x.view(3, 20, D), x.view(3, 20, D).transpose(0, 1).contiguous().transpose(0, 1)]
    ws = [w, ww[:, :D], w.t().contiguous().t(), wo[1:].view(V, D), w.repeat_interleave(2, 0)[::2]]
    for i, xv in enumerate(xs):
        for wv in ws if i == 0 else ws[:1]:
            xl, wl = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
            yv = y.view(xv.shape[:-1]).to([torch.int64, torch.int32, torch.int16][i % 3])
            got = lm_head.linear_cross_entropy(xl, wl, yv)
            assert (got.detach().double() - loss).abs() <= ltol
            a, b = torch.autograd.grad(got, [xl, wl])
            near(a, dx, dxt, dt, V + D)
            near(b, dw, dwt, dt, T + D)
    rows = lm_head.linear_cross_entropy(xs[3], w, y.view(3, 20), reduction="none")
    assert rows.shape == (3, 20)
    # a token's row repeated (rows that overlap)
    one = x[:1].expand(T, D)
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(one, w, y, reduction="sum")
    xl, wl = one.detach().requires_grad_(True), w.clone().requires_grad_(True)
    got = lm_head.linear_cross_entropy(xl, wl, y, reduction="sum")
    a, b = torch.autograd.grad(got, [xl, wl])
    near(a, dx, dxt, dt, V + D)
    near(b, dw, dwt, dt, T + D)
    # a single token without a batch dimension
    got = lm_head.linear_cross_entropy(x[0], w, y[0].abs().clamp(max=V - 1), reduction="none")
    assert got.shape == ()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 256])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_few_rows_are_rounded_once(dev, T, dt, reduction):
    """With few rows the targets' part of the gradients is as near as one rounding allows."""
    V, D = 1000, 128
    g = torch.Generator().manual_seed(T)
    y = torch.randperm(V, generator=g)[:T].to(dev)
    x = torch.randn(T, D, generator=g).to(DT[dt]).to(dev).requires_grad_()
    w = torch.zeros(V, D)
    w[y.cpu()] = torch.randn(T, D, generator=g) * 0.3
    w = w.to(DT[dt]).to(dev).requires_grad_()
    gr = torch.randn(T, generator=g).to(dev) if reduction == "none" else torch.tensor(0.7, device=dev)
    loss = lm_head.linear_cross_entropy(x, w, y, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), gr)
    x64, w64 = x.detach().double(), w.detach().double()
    p = (x64 @ w64.T).softmax(-1)
    g64 = gr.double().expand(T)[:, None]
    at = torch.nn.functional.one_hot(y, V).double()
    dz, other = g64 * (p - at), (g64 * p).abs() * (1 - at)
    # the other entries of dz are rounded (fp16: or lie under its steps below 2^-14, 2^-24 of the largest
    # row's 2^-15), the sums are fp32: 1000 terms of 2^-24 of the products' absolute sum
    half = torch.finfo(DT[dt]).eps / 2
    tiny = 2 ** -38 * g64.abs().max()
    for got, want, off, total in ((dx, dz @ w64, (other * half + tiny) @ w64.abs(), dz.abs() @ w64.abs()),
                                  (dw, dz.T @ x64, (other * half + tiny).T @ x64.abs(), dz.abs().T @ x64.abs())):
        # (2^-25: half of fp16's last step)
        bound = want.abs() * half * 1.001 + off * 1.01 + total * 1000 * 2 ** -24 + 2 ** -25
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("gap", [0.0, 10.0, 40.0, -40.0])
def test_sure_rows(dev, dt, gap):
    """Few rows whose target is nearly sure, or nearly impossible, some with a gradient of 0 or far below the others'."""
    T, V, D = 5, 600, 64
    g = torch.Generator().manual_seed(3)
    x = torch.zeros(T, D)
    x[:, 0] = 8
    x[:, 1:] = torch.randn(T, D - 1, generator=g) * 0.1
    w = torch.randn(V, D, generator=g) * 0.1
    w[:, 0] = 0
    y = torch.arange(T) * 7
    w[y[0], 0] = gap / 8  # the first row's target for all rows
    y[1:3] = y[0]
    x, w = (t.to(DT[dt]).to(dev).requires_grad_() for t in (x, w))
    y, gr = y.to(dev), torch.tensor([1.0, 0.0, -1e-6, 0.5, 1e-12], device=dev)
    loss = lm_head.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), gr)
    x64, w64, g64 = x.detach().double(), w.detach().double(), gr.double()[:, None]
    p = (x64 @ w64.T).softmax(-1)
    dz = g64 * (p - torch.nn.functional.one_hot(y, V).double())
    # an entry of dz: rounded (fp16: to steps of 2^-38 of the largest); p and p - 1 in fp32, whose exponentials'
    # arguments, up to 45, are off by 2^-22 of themselves from the sums of 64 products and the scaling: 2^-16
    half = torch.finfo(DT[dt]).eps / 2
    off = dz.abs() * (half + 2 ** -16) + g64.abs() * (p * 2 ** -16).clamp(max=2 ** -20) + 2 ** -38
    for got, want, o in ((dx, dz @ w64, off @ w64.abs()), (dw, dz.T @ x64, off.T @ x64.abs())):
        bound = want.abs() * (half * 1.001 + 600 * 2 ** -24) + o * 1.01 + 2 ** -25
        assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 65])
def test_a_single_row_whose_stride_is_not_its_width(dev, D):
    """One token, and a vocabulary of one: a transposed column's only row has a stride of 1."""
    x = torch.randn(D, 1, device=dev).to(torch.bfloat16).t()
    w = torch.randn(D, 1, device=dev).to(torch.bfloat16).t()
    y = torch.zeros(1, dtype=torch.int64, device=dev)
    assert x.stride(0) == w.stride(0) == 1
    many = torch.randn(37, D, device=dev).to(torch.bfloat16)
    for a, b, t in ((x, many, y + 5), (many, w, y.expand(37)), (x, w, y)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        a64, b64 = a.detach().double().requires_grad_(), b.detach().double().requires_grad_()
        loss = lm_head.linear_cross_entropy(a, b, t, reduction="sum")
        want = torch.nn.functional.cross_entropy(a64 @ b64.T, t, reduction="sum")
        da, db = torch.autograd.grad(loss, (a, b))
        wa, wb = torch.autograd.grad(want, (a64, b64))
        # (65 products of up to 4 x 4 summed in fp32; exponentials, one more sum and a logarithm)
        assert abs(loss.item() - want.item()) <= 2e-5 * max(1.0, abs(want.item()))
        # the gradient of the logits and each gradient are rounded once, by up to 2^-8 of itself; sums of up
        # to 37 terms of at most 4.5, and fp32's part below
        for g, r in ((da, wa), (db, wb)):
            bound = 2 ** -8 * r.abs() + 37 * 4.5 * 2 ** -8 + 1e-4
            assert g.shape == r.shape and ((g.double() - r).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_no_tokens(dev, dt):
    w = torch.randn(50, 64, device=dev).to(DT[dt]).requires_grad_(True)
    x = torch.empty(0, 64, device=dev, dtype=DT[dt], requires_grad=True)
    y = torch.empty(0, dtype=torch.int64, device=dev)
    assert torch.isnan(lm_head.linear_cross_entropy(x, w, y))
    assert lm_head.linear_cross_entropy(x, w, y, reduction="none").shape == (0,)
    loss = lm_head.linear_cross_entropy(x, w, y, reduction="sum")
    assert loss.item() == 0.0
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert dx.shape == (0, 64) and (dw == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_gradients_far_from_one(dev, dt, reduction):
    """A loss scaled up or averaged over very many rows, and rows whose gradients differ widely."""
    x, w, y, g = make(64, 400, 64, dt, 0.0, dev)
    for size in (2.0 ** -18, 1.0, 2.0 ** 6):
        grad = torch.tensor(size, device=dev)
        if reduction == "none":
            grad = (torch.randn(64, generator=g).exp2() * size).to(dev)
        _, (dx, dxt), (dw, dwt) = reference(x, w, y, reduction=reduction, grad=grad)
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        a, b = torch.autograd.grad(lm_head.linear_cross_entropy(xl, wl, y, reduction=reduction), [xl, wl], grad)
        near(a, dx, dxt, dt, 464)
        near(b, dw, dwt, dt, 128)
    # a gradient expanded over the rows, and one of zeros
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    rows = lm_head.linear_cross_entropy(xl, wl, y, reduction="none")
    _, (dx, dxt), (dw, dwt) = reference(x, w, y, reduction="none")
    a, b = torch.autograd.grad(rows.sum(), [xl, wl], retain_graph=True)
    near(a, dx, dxt, dt, 464)
    near(b, dw, dwt, dt, 128)
    a, b = torch.autograd.grad(rows, [xl, wl], torch.zeros_like(rows))
    assert (a == 0).all() and (b == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_large_logits_do_not_overflow(dev, dt):
    x = torch.zeros(8, 64, device=dev, dtype=DT[dt])
    w = torch.zeros(300, 64, device=dev, dtype=DT[dt])
    x[:, 0] = 100.0
    w[:, 0] = torch.linspace(-100, 100, 300, device=dev).to(DT[dt])
    y = torch.tensor([0, 299, 298, 150, 1, 299, 299, 2], device=dev)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    rows = lm_head.linear_cross_entropy(xl, wl, y, reduction="none")
    z = x.detach().double() @ w.detach().double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    # logits of 10^4 are exact here (one product each): the loss is fp32's rounding of 2 * 10^4
    assert ((rows.detach().double() - want).abs() <= 4 * U * 2e4).all()
    a, b = torch.autograd.grad(rows.sum(), [xl, wl])
    assert torch.isfinite(a).all() and torch.isfinite(b).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_gradient_against_differences(dev, dt):
    x, w, y, g = make(6, 50, 70, dt, 0.0, dev)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(lm_head.linear_cross_entropy(xl, wl, y), [xl, wl])

    def value(x, w):
        return F.cross_entropy(x @ w.t(), y).item()

    xd, wd = x.double(), w.double()
    h = 1e-5  # the difference's own error is about h^2 = 1e-10 and 1e-15 / h = 1e-10
    for t, d in ((0, 0), (3, 69), (5, 33)):
        a, b = xd.clone(), xd.clone()
        a[t, d] += h
        b[t, d] -= h
        want = (value(a, wd) - value(b, wd)) / (2 * h)
        assert abs(dx[t, d].item() - want) <= 3 * STEP[dt] * dx[t].abs().max().item() + 1e-6
    for v, d in ((int(y[0]), 0), (49, 69), (int(y[3]), 33)):
        a, b = wd.clone(), wd.clone()
        a[v, d] += h
        b[v, d] -= h
        want = (value(xd, a) - value(xd, b)) / (2 * h)
        assert abs(dw[v, d].item() - want) <= 3 * STEP[dt] * dw.abs().max().item() + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_repeat_stream_and_graph(dev, dt):
    T, V, D = 700, 3000, 200
    x, w, y, g = make(T, V, D, dt, 0.3, dev)

    def step(x, w, y):
        loss = lm_head.linear_cross_entropy(x, w, y)
        return (loss, *torch.autograd.grad(loss, [x, w]))

    def leaves():
        return x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    want = [t.detach().clone() for t in step(*leaves(), y)]
    assert all(torch.equal(a, b) for a, b in zip(want, step(*leaves(), y)))
    lv = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*lv, y)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got, lv
    sx, sw = torch.zeros_like(x).requires_grad_(True), torch.zeros_like(w).requires_grad_(True)
    sy = torch.zeros_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sw, sy)
    for r in range(3):  # other inputs, and another number of ignored rows, each time
        yr = torch.where(torch.rand(T, generator=g).to(dev) < 0.3 * r, -100, y.clamp(min=0).roll(r))
        with torch.no_grad():
            sx.copy_(x.roll(r, 0))
            sw.copy_(w.roll(r, 0))
            sy.copy_(yr)
        graph.replay()
        torch.cuda.synchronize()
        want = step(x.roll(r, 0).requires_grad_(True), w.roll(r, 0).requires_grad_(True), yr)
        assert all(torch.equal(a, b) for a, b in zip(want, out)), r


@pytest.mark.gpu
def test_compiles(dev):
    x, w, y, g = make(100, 400, 100, "bf16", 0.2, dev)

    def step(x, w):
        return lm_head.linear_cross_entropy(x * 2, w, y) + lm_head.linear_cross_entropy(x, w, y, reduction="none").sum()

    grads = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = f(xl, wl)
        grads.append((loss.detach(), *torch.autograd.grad(loss, [xl, wl])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    for D in (100, 128):
        x, w, y, g = make(50, 300, D, "bf16", 0.2, dev)
        torch.library.opcheck(torch.ops.cinnamon_amd.linear_ce_forward, (x, w, y, -100, 2),
                              test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_a_model_step_with_tied_heads(dev):
    """Main and next-but-one losses over one tied weight, as the training step composes them, with
    gradients through a norm, against the same step on plain logits in 64 bits."""
    torch.manual_seed(5)
    B, L, D, V = 2, 65, 128, 1000
    emb = torch.randn(V, D, device=dev) * 0.05
    ids = torch.randint(0, V, (B, L + 1), device=dev)
    mix = torch.randn(D, D, device=dev) / math.sqrt(D)

    def step(emb, mix, loss_of):
        h = F.embedding(ids[:, :-1], emb) @ mix
        h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + 1e-6)
        main = loss_of(h, emb, ids[:, 1:])
        mtp = loss_of(h[:, :-1], emb, ids[:, 2:])
        return main + 0.3 * mtp

    ref = [t.double().requires_grad_(True) for t in (emb, mix)]
    want = step(*ref, lambda h, w, y: F.cross_entropy((h @ w.t()).reshape(-1, V), y.reshape(-1)))
    dwant = torch.autograd.grad(want, ref)
    got = [t.clone().requires_grad_(True) for t in (emb, mix)]
    loss = step(*got, lm_head.linear_cross_entropy)
    dgot = torch.autograd.grad(loss, got)
    # fp32 throughout: sums of at most 1000 terms in each of three chained products
    assert abs(loss.item() - want.item()) <= 3 * math.sqrt(1000) * U * want.item()
    for a, b in zip(dgot, dwant):
        assert (a - b).norm() <= 12 * math.sqrt(1000) * U * b.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,V,D", [(16, 700, 64), (128, 1500, 96), (129, 1500, 96), (300, 3001, 130), (2100, 900, 64)])
@pytest.mark.parametrize("value", ["lowest", "-inf"])
def test_masked_entries_of_the_vocabulary(dev, dt, T, V, D, value):
    """Entries whose weight holds the type's lowest value or -inf at a constant feature: as if the
    vocabulary had no such entries, at any number of rows.  With -inf, 0 * inf makes that feature's gradient of x NaN."""
    low = -math.inf if value == "-inf" else torch.finfo(DT[dt]).min
    x, w, y, g = make(T, V, D, dt, 0.1, dev)
    x[:, 5] = 1.0
    gone = torch.zeros(V, dtype=torch.bool)
    gone[torch.randperm(V, generator=g)[:9]] = True
    gone[-1] = True
    gone[y[y >= 0].cpu()] = False
    assert gone.any()
    gone = gone.to(dev)
    w[gone, 5] = low
    y2 = torch.where(y >= 0, torch.cumsum(~gone, 0)[y.clamp(min=0)] - 1, y)
    grad = torch.randn(T, generator=g).to(dev)
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w[~gone], y2, reduction="none", grad=grad)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    with torch.no_grad():
        plain = lm_head.linear_cross_entropy(x, w, y, reduction="none")
    got = lm_head.linear_cross_entropy(xl, wl, y, reduction="none")
    assert torch.isfinite(got).all() and torch.equal(plain, got.detach())
    assert ((got.detach().double() - loss).abs() <= ltol).all()
    a, b = torch.autograd.grad(got, [xl, wl], grad)
    assert (b[gone] == 0).all()
    near(b[~gone], dw, dwt, dt, T + D)
    if value == "-inf":
        assert torch.isnan(a[y >= 0][:, 5]).all()
        keep = torch.arange(D, device=dev) != 5
        a, dx, dxt = a[:, keep], dx[:, keep], dxt[:, keep]
    near(a, dx, dxt, dt, V + D)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [100, 200])
def test_infinities_of_fp32_rows(dev, T):
    """What an infinity or NaN makes of a row's loss does not depend on the number of rows: one row of x
    holds it, the others' losses and gradients stay."""
    x, w, y, g = make(T, 1000, 72, "fp32", 0.0, dev)
    w[:, 7] = w[:, 7].abs() + 0.1
    w[0, 7] = 0.2
    want = lm_head.linear_cross_entropy(x, w, y, reduction="none")
    for value, loss in ((math.inf, "nan"), (-math.inf, "nan"), (math.nan, "nan"), (torch.finfo(torch.float32).max, "any")):
        z = x.clone()
        z[3, 7] = value
        leaf, wl = z.clone().requires_grad_(True), w.clone().requires_grad_(True)
        got = lm_head.linear_cross_entropy(leaf, wl, y, reduction="none")
        others = torch.arange(T, device=dev) != 3
        assert torch.equal(got[others].detach(), want[others])
        if loss == "nan":
            assert torch.isnan(got[3])
        (dx,) = torch.autograd.grad(got[others].sum(), [leaf])
        assert torch.isfinite(dx[others]).all()
    # every entry of the vocabulary at -inf for a row: 0 / 0, as in the softmax itself
    z = x.clone()
    z[3, 7] = -math.inf
    assert torch.isnan(lm_head.linear_cross_entropy(z, w, y, reduction="none")[3])
    # a target at -inf: its loss is inf, and the gradient pushes away from all the others
    v = w.clone()
    x[:, 5] = 1.0
    v[y[0], 5] = -math.inf
    leaf = v.requires_grad_(True)
    rows = lm_head.linear_cross_entropy(x, leaf, y, reduction="none")
    of = y == y[0]
    assert torch.isposinf(rows[of]).all() and torch.isfinite(rows[~of]).all()
    (dw,) = torch.autograd.grad(rows.sum(), [leaf])
    assert torch.isfinite(dw).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,V,D", [(1, 777, 40), (32, 3001, 128), (100, 1500, 64), (128, 2049, 300)])
def test_kept_logits_and_logits_formed_again(dev, monkeypatch, dt, T, V, D):
    """Either way gives the gradients; the same ones where the logits are summed in the same order."""
    x, w, y, g = make(T, V, D, dt, 0.1, dev)
    grad = torch.randn(T, generator=g).to(dev)
    _, (dx, dxt), (dw, dwt) = reference(x, w, y, reduction="none", grad=grad)
    losses = []
    for kept in (True, False):
        monkeypatch.setattr(lm_head, "_keeps", lambda T, D, dtype: kept)
        lm_head._sizes.cache_clear()
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = lm_head.linear_cross_entropy(xl, wl, y, reduction="none")
        a, b = torch.autograd.grad(loss, [xl, wl], grad)
        near(a, dx, dxt, dt, V + D)
        near(b, dw, dwt, dt, T + D)
        losses.append(loss.detach())
    lm_head._sizes.cache_clear()
    assert torch.equal(*losses)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_kept_logits_are_fewer_bytes_than_the_weight(dt):
    """Written and read they are no more than the weight that gives them again."""
    dtype, es = DT[dt], DT[dt].itemsize
    V = 131072
    for D in (8, 64, 128, 256, 512, 1024, 4096):
        for T in (1, 2, 16, 31, 64, 128, 129, 1000):
            state = lm_head._layout(T, D, V, dtype)[1]
            wide = -(-D // 64) * 64
            rest = 3 * T * wide * es + 64 * T + 4096  # x's copy and the words a row
            if dtype == torch.float32 and T > 128:
                rest += 6 * V * wide                  # the weight's, in three parts or padded
            elif wide != D:
                rest += V * wide * es
            assert state <= rest + V * D * es // 2, (D, T)
    assert lm_head._layout(16, 1024, V, dtype)[1] >= 4 * 16 * V


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(257, 1000, 128), (700, 20000, 200), (1100, 17001, 64), (5000, 16500, 136), (9000, 16400, 64)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("spread", ["all", "few", "one"])
def test_many_rows_keep_their_targets_entries(dev, T, V, D, dt, reduction, spread):
    """What rounding takes off an entry of dz at a target comes back in both gradients: any number of rows with
    the same target, some ignored."""
    g = torch.Generator().manual_seed(T)
    y = {"all": torch.randint(0, V, (T,), generator=g), "few": torch.randint(0, 9, (T,), generator=g) * (V // 9),
         "one": torch.full((T,), V - 1)}[spread]
    x = torch.randn(T, D, generator=g) * 0.3
    w = torch.randn(V, D, generator=g) * 0.3
    y[torch.rand(T, generator=g) < 0.1] = -100
    x, w = (t.to(DT[dt]).to(dev).requires_grad_() for t in (x, w))
    y = y.to(dev)
    gr = torch.randn(T, generator=g).to(dev) if reduction == "none" else torch.tensor(0.7, device=dev)
    loss = lm_head.linear_cross_entropy(x, w, y, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), gr)
    x64, w64 = x.detach().double(), w.detach().double()
    kept = (y >= 0)[:, None]
    p = (x64 @ w64.T).softmax(-1)
    g64 = (gr.double().expand(T)[:, None] / (1 if reduction == "none" else kept.sum())) * kept
    at = torch.nn.functional.one_hot(y.clamp(min=0), V).double()
    dz, other, mine = g64 * (p - at), (g64 * p).abs() * (1 - at), (g64 * (p - at) * at).abs()
    # The other entries are rounded (fp16: or lie under its steps, 2^-24 of the largest row's 2^-15), the
    # targets' are held to 2 half steps of half a step; p is off by the sums' D 2^-24 of products up to 0.3^2 D 6
    # and 2^-18; the sums are fp32 chains of K / 32 groups of 32 products and at most 256 slabs
    half = torch.finfo(DT[dt]).eps / 2
    tiny = 2 ** -38 * g64.abs().max()
    off = other * half + mine * 2 * half * half + (g64 * p).abs() * (D * 2 ** -24 * 0.6 * D + 2 ** -18) + tiny * kept
    for got, want, o, total, K in ((dx, dz @ w64, off @ w64.abs(), dz.abs() @ w64.abs(), V),
                                   (dw, dz.T @ x64, off.T @ x64.abs(), dz.abs().T @ x64.abs(), T)):
        bound = want.abs() * half * 1.001 + o * 1.01 + total * (K / 32 + 300) * 2 ** -24 + 2 ** -25
        d = (got.double() - want).abs()
        assert (d <= bound).all(), (d / bound).max()


@pytest.mark.gpu
def test_masked_entries_of_a_later_piece(dev):
    """fp32, two pieces of the vocabulary, a masked entry in each."""
    T, V, D = 9000, 35001, 64
    x, w, y, g = make(T, V, D, "fp32", 0.1, dev)
    x[:, 5] = 1.0
    gone = torch.zeros(V, dtype=torch.bool, device=dev)
    gone[[10, V - 3]] = True
    y[(y == 10) | (y == V - 3)] = 0
    w[gone, 5] = -math.inf
    y2 = torch.where(y >= 0, torch.cumsum(~gone, 0)[y.clamp(min=0)] - 1, y)
    grad = torch.tensor(0.7, device=dev)
    (loss, ltol), (dx, dxt), (dw, dwt) = reference(x, w[~gone], y2, reduction="sum", grad=grad)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = lm_head.linear_cross_entropy(xl, wl, y, reduction="sum")
    assert abs(got.item() - loss.item()) <= ltol.item()
    a, b = torch.autograd.grad(got, [xl, wl], grad)
    assert (b[gone] == 0).all()
    near(b[~gone], dw, dwt, "fp32", T + D)
    keep = torch.arange(D, device=dev) != 5
    near(a[:, keep], dx[:, keep], dxt[:, keep], "fp32", V + D)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_a_graph_whose_weight_is_masked_in_some_replays(dev, dt):
    T, V, D = 300, 2000, 128
    x, w, y, g = make(T, V, D, dt, 0.2, dev)
    x[:, 5] = 1.0
    masked = w.clone()
    masked[[3, 700, 1999], 5] = -math.inf

    def step(x, w):
        loss = lm_head.linear_cross_entropy(x, w, y, reduction="none")
        return (loss, *torch.autograd.grad(loss.sum(), [x, w]))

    def leaves(w):
        return x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    step(*leaves(w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    sx, sw = leaves(w)
    with torch.cuda.graph(graph):
        out = step(sx, sw)
    for v in (w, masked, w, masked, masked, w):
        with torch.no_grad():
            sw.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*leaves(v))
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 64, 128])
def test_long_fp32_sums(dev, T):
    """Logits of 4096 products.  A rounding of a sum s is off by u |s| / sqrt(3) in the mean square at most; the sum of
    k products of variance v has mean square k v.  Sums of 32 products each, then of the 128 of them:
    u sqrt(v) times 32 sqrt(128 / 6) and 128 sqrt(32 / 6), 150 and 300 (one after the other all the way: 4096 / sqrt(6) =
    1670).  Their root of squares here, 0.3 of it more for the few rows, and two roundings of the loss itself."""
    D = 4096
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, D, generator=g)
    w = torch.zeros(2, D)
    w[0] = torch.randn(D, generator=g)
    x = torch.where((x @ w[0])[:, None] < 0, -x, x).to(dev)   # the first logit positive, the second one 0
    w = w.to(dev)
    loss = lm_head.linear_cross_entropy(x, w, torch.ones(T, dtype=torch.int64, device=dev), reduction="none")
    z = x.double() @ w[0].double()
    want = torch.nn.functional.softplus(z, threshold=1e9)
    rms = (loss.double() - want).square().mean().sqrt()
    v = (x.double() * w[0].double()).square().mean().sqrt()
    assert rms <= 1.3 * math.hypot(150, 300) * U * v + 2 * U * z.square().mean().sqrt()


def test_refusals():
    with FakeTensorMode():
        def fake(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        i64 = torch.int64
        x, w, y = fake(4, 64), fake(100, 64), fake(4, dtype=i64)
        f = lm_head.linear_cross_entropy
        for bad in [
            lambda: f(torch.empty(4, 64, dtype=torch.bfloat16), w, y),
            lambda: f(x, torch.empty(100, 64, dtype=torch.bfloat16), y),
            lambda: f(x, w, torch.zeros(4, dtype=i64)),
            lambda: f(x, fake(100, 32), y),
            lambda: f(x, fake(100, 64, 1), y),
            lambda: f(x, w, fake(5, dtype=i64)),
            lambda: f(x, w, fake(4, 1, dtype=i64)),
            lambda: f(x, fake(100, 64, dtype=torch.float32), y),
            lambda: f(fake(4, 64, dtype=torch.float64), fake(100, 64, dtype=torch.float64), y),
            lambda: f(x, w, fake(4, dtype=torch.float32)),
            lambda: f(x, w, fake(4, dtype=torch.bool)),
            lambda: f(x, w, y, reduction="max"),
            lambda: f(x, fake(0, 64), y),
            lambda: f(fake(4, 0), fake(100, 0), y),
        ]:
            with pytest.raises(AssertionError):
                bad()
        assert f(x, w, y).shape == () and f(x, w, y).dtype == torch.float32
        assert f(fake(2, 2, 65), fake(100, 65), fake(2, 2, dtype=i64), reduction="none").shape == (2, 2)


_FWD = [16, 0, 4, 64, 64, 16, 100, 64, 16, -100, 1, 16, None, 16, 16, 16, 16, 16, 1 << 30, None, None]
_BWD = [16, 0, 4, 64, 16, 100, 64, 16, 16, 16, 0, 1, 16, 16, 16, 1 << 30, None, None]


@pytest.mark.parametrize("name,ok,at,value", [
    ("cin_linear_ce_forward", _FWD, 1, 4), ("cin_linear_ce_forward", _FWD, 2, -1), ("cin_linear_ce_forward", _FWD, 3, 0),
    ("cin_linear_ce_forward", _FWD, 3, 1 << 19), ("cin_linear_ce_forward", _FWD, 4, 63), ("cin_linear_ce_forward", _FWD, 6, 0),
    ("cin_linear_ce_forward", _FWD, 7, 63), ("cin_linear_ce_forward", _FWD, 7, 65), ("cin_linear_ce_forward", _FWD, 5, 20),
    ("cin_linear_ce_forward", _FWD, 0, None), ("cin_linear_ce_forward", _FWD, 8, None), ("cin_linear_ce_forward", _FWD, 11, None),
    ("cin_linear_ce_forward", _FWD, 13, None), ("cin_linear_ce_forward", _FWD, 17, None), ("cin_linear_ce_forward", _FWD, 18, 10),
    ("cin_linear_ce_backward", _BWD, 1, 4), ("cin_linear_ce_backward", _BWD, 2, 0), ("cin_linear_ce_backward", _BWD, 6, 65),
    ("cin_linear_ce_backward", _BWD, 4, 18), ("cin_linear_ce_backward", _BWD, 9, None), ("cin_linear_ce_backward", _BWD, 10, -1),
    ("cin_linear_ce_backward", _BWD, 14, None), ("cin_linear_ce_backward", _BWD, 15, 100), ("cin_linear_ce_backward", _BWD, 3, 65),
    # launches of 2^32 threads, and pointers that 16-byte accesses do not fit
    ("cin_linear_ce_forward", _FWD, 2, 1 << 26), ("cin_linear_ce_forward", _FWD, 6, (1 << 29) + 1),
    ("cin_linear_ce_forward", _FWD, 11, 24), ("cin_linear_ce_forward", _FWD, 12, 24), ("cin_linear_ce_forward", _FWD, 17, 24),
    ("cin_linear_ce_backward", _BWD, 0, 24), ("cin_linear_ce_backward", _BWD, 12, 24), ("cin_linear_ce_backward", _BWD, 14, 24),
    ("cin_linear_ce_forward", _FWD, 19, 24), ("cin_linear_ce_backward", _BWD, 16, 24),
])
def test_c_refusals(name, ok, at, value):
    args = list(ok)
    args[at] = value
    with pytest.raises(ValueError):
        _lib.call(name, *args)


def test_workspace_grows_with_the_call_and_is_bounded():
    ws = _lib.load().cin_linear_ce_workspace
    assert ws(0, -1, 64, 100, 1) == -1 and ws(0, 4, 64, 100, 0) > 0
    for T, D, V in ((1, 64, 100), (8192, 4096, 131072), (100000, 1024, 200000)):
        # a piece of the logits' gradient, and partial sums of x's gradient
        assert 0 < ws(0, T, D, V, 1) <= (1 << 30) + T * 1024 + 256 * 2 * T + 4 * T * D * 4 + (256 << 20)
