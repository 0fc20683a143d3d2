"""lm_head.verify_drafts against its definition (GPU for the operator, CPU for the refusals).

The operator's sums are in 64 bits, in another order than the definition's: a border between two tokens
moves by at most V 2^-53 of the whole (1.5e-11 at 131072), so a random number lies between the two in one draw of 1e5 at
most; in the cases here the uniform numbers keep a margin of 1e-9 of the whole from every border.
"""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from cinnamon_amd import _lib, lm_head

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def definition(tokens, q, p, u, counts=None):
    """(tokens, accepted, the least distance of a deciding number from its border) in 64 bits."""
    tokens, p, u = tokens.cpu(), p.double().cpu(), u.double().cpu()
    B, K = tokens.shape
    V = p.shape[2]
    if q is None:
        q = torch.zeros(B, K, V, dtype=torch.float64)
        for b in range(B):
            for i in range(K):
                if 0 <= tokens[b, i] < V:
                    q[b, i, tokens[b, i]] = 1.0
        certain = True
    else:
        q, certain = q.double().cpu(), False
    out, accepted, margin = torch.full((B, K + 1), -1), torch.zeros(B, dtype=torch.int64), 1.0
    for b in range(B):
        limit = K if counts is None else min(max(int(counts[b]), 0), K)
        n = 0
        while n < limit:
            x = int(tokens[b, n])
            if not 0 <= x < V or not bool(u[b, n] * q[b, n, x] < p[b, n, x]):
                break
            out[b, n] = x
            n += 1
        whole = p[b, n].clamp_min(0)
        rest = (p[b, n] - q[b, n]).clamp_min(0) if n < limit else whole
        if certain and n < limit and 0 <= tokens[b, n] < V:
            rest[tokens[b, n]] = 0
        if rest.sum() == 0:
            rest = whole
        cum = rest.cumsum(0)
        accepted[b] = n
        if not (cum[-1] > 0 and cum[-1] < math.inf):
            continue
        target = u[b, K] * cum[-1]
        margin = min(margin, float(((cum - target).abs() / cum[-1]).min()))
        hits = ((cum > target) & (rest > 0)).nonzero()
        out[b, n] = hits[0, 0] if len(hits) else rest.nonzero()[-1, 0]
    return out, accepted, margin


def inputs(dev, B, K, V, dt, seed=1, near=0.7):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, K + 1, V, generator=g) * 2
    p = torch.softmax(z, -1)
    q = torch.softmax(z[:, :K] + near * torch.randn(B, K, V, generator=g), -1)
    tokens = torch.multinomial(q.reshape(B * K, V), 1, generator=g).view(B, K) if K else torch.zeros(B, 0, dtype=torch.int64)
    u = torch.rand(B, K + 1, generator=g)
    return tokens.to(dev), q.to(DT[dt]).to(dev), p.to(DT[dt]).to(dev), u.to(dev)


def check(got, want):
    assert want[2] > 1e-9, "the case's numbers lie on a border"
    assert got[0].dtype == got[1].dtype == torch.int64
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 0, 7), (3, 2, 2), (1, 1, 32000), (17, 7, 5025), (5, 63, 77), (40, 3, 2048), (9, 4, 2049),
                                   (2, 2, 40001)])
def test_against_the_definition(dev, B, K, V, dt):
    for seed in range(3):
        tokens, q, p, u = inputs(dev, B, K, V, dt, seed)
        check(lm_head.verify_drafts(tokens, q, p, u), definition(tokens, q, p, u))
        check(lm_head.verify_drafts(tokens, None, p, u), definition(tokens, None, p, u))
        counts = torch.randint(-1, K + 2, (B,), generator=torch.Generator().manual_seed(seed)).to(dev)
        check(lm_head.verify_drafts(tokens, q, p, u.double(), counts), definition(tokens, q, p, u, counts))
        # equal rows: every token is kept, and the last is drawn
        same = p[:, :K]
        got = lm_head.verify_drafts(tokens, same, p, u)
        kept = (same.gather(2, tokens[..., None])[..., 0] > 0).long().cumprod(1).sum(1)
        assert torch.equal(got[1], kept)
        check(got, definition(tokens, same, p, u))


@pytest.mark.gpu
def test_a_large_vocabulary_in_parts(dev):
    """Every part of a row is drawn from, its first and last tokens too."""
    V = 131072
    p = torch.zeros(64, 1, V, device=dev)
    at = torch.arange(64, device=dev) * 2048 + torch.tensor([0, 2047, 1, 1000], device=dev).repeat(16)
    p[torch.arange(64, device=dev), 0, at] = 0.25
    u = torch.rand(64, 1, generator=torch.Generator().manual_seed(1)).to(dev)
    tokens, n = lm_head.verify_drafts(torch.empty(64, 0, dtype=torch.int64, device=dev), None, p, u)
    assert torch.equal(tokens[:, 0], at) and (n == 0).all()
    # two tokens of equal weight far apart, numbers on both sides and on the border (which belongs to the second)
    p = torch.zeros(3, 1, V, device=dev)
    p[:, 0, 5] = p[:, 0, V - 1] = 0.5
    u = torch.tensor([[0.49], [0.5], [0.51]], device=dev)
    tokens, _ = lm_head.verify_drafts(torch.empty(3, 0, dtype=torch.int32, device=dev), None, p, u)
    assert tokens[:, 0].tolist() == [5, V - 1, V - 1]


@pytest.mark.gpu
def test_borders_and_rows_with_nothing(dev):
    V = 100
    p, q = torch.zeros(9, 2, V, device=dev), torch.zeros(9, 1, V, device=dev)
    p[:, :, 3], p[:, :, 90] = 0.5, 0.5
    q[:, 0, 3] = 1.0
    tokens = torch.full((9, 1), 3, device=dev)
    u = torch.full((9, 2), 0.25, device=dev)
    u[0, 0] = 0.5                      # u q = p: not kept, the rest is token 90
    u[1, 0] = 0.5 - 2 ** -25           # just kept
    u[2, 0], p[2, 0, 90], p[2, 0, 3] = 0.9, 0, 0.5  # not kept, and nothing of p above q: from p itself
    tokens[3], tokens[4] = -1, V       # tokens outside: not kept, the rest drawn
    p[5, 1] = 0                        # kept, then a row with nothing
    p[6, 1, 7] = math.nan
    p[7, 1, 7] = math.inf
    q[8, 0] = 0                        # a draft that its own probabilities exclude: kept where p has it
    u[8, 1] = 1.0                      # a number out of range: the last token with any probability
    out, n = lm_head.verify_drafts(tokens, q, p, u)
    assert n.tolist() == [0, 1, 0, 0, 0, 1, 1, 1, 1]
    assert out.tolist() == [[90, -1], [3, 3], [3, -1], [90, -1], [90, -1], [3, -1], [3, -1], [3, -1], [3, 90]]


@pytest.mark.gpu
def test_strides_and_offsets_past_32_bits(dev):
    B, K, V = 3, 2, 1001
    tokens, q, p, u = inputs(dev, B, K, V, "bf16", 5)
    want = definition(tokens, q, p, u)
    wide = torch.zeros(B, K + 2, V + 5, dtype=p.dtype, device=dev)
    wide[:, 1:, 3:-2] = p
    check(lm_head.verify_drafts(tokens, q, wide[:, 1:, 3:-2], u), want)
    across = q.transpose(1, 2).contiguous().transpose(1, 2)
    many = torch.zeros(K, 2 * B, dtype=torch.int32, device=dev)
    many[:, ::2] = tokens.t()
    ut = torch.zeros(K + 1, B, device=dev)
    ut.copy_(u.t())
    counts = torch.tensor([9, 2, 9, 1, 9, 2], device=dev)[1::2]
    check(lm_head.verify_drafts(many[:, ::2].t(), across, p, ut.t(), counts), definition(tokens, q, p, u, counts))
    step = (1 << 31) + 64  # elements from one sequence to the next
    far = torch.zeros(2 * step + 3 * V, dtype=torch.bfloat16, device=dev)
    view = torch.as_strided(far, (B, K + 1, V), (step, V, 1))
    view.copy_(p)
    check(lm_head.verify_drafts(tokens, q, view, u), want)


@pytest.mark.gpu
def test_distribution(dev):
    """Kept or drawn, a position's token has the target's probabilities: 2^16 sequences of one draft, counts within
    six standard deviations."""
    B, V = 1 << 16, 12
    g = torch.Generator().manual_seed(8)
    p = torch.softmax(torch.randn(V, generator=g), 0)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    tokens = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1)
    u = torch.rand(B, 2, generator=g)
    out, _ = lm_head.verify_drafts(tokens.to(dev), q.to(dev).expand(B, 1, V), p.to(dev).expand(B, 2, V), u.to(dev))
    n = torch.bincount(out[:, 0].cpu(), minlength=V).double()
    assert ((n - B * p.double()).abs() <= 6 * (B * p.double() * (1 - p.double())).sqrt()).all()


@pytest.mark.gpu
def test_streams_graphs_and_no_sequences(dev):
    tokens, q, p, u = inputs(dev, 6, 3, 5000, "fp32", 9)
    eager = lm_head.verify_drafts(tokens, q, p, u)
    out, n = lm_head.verify_drafts(tokens[:0], q[:0], p[:0], u[:0])
    assert out.shape == (0, 4) and n.shape == (0,)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = lm_head.verify_drafts(tokens, q, p, u)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lm_head.verify_drafts(tokens, q, p, u)
    for seed in range(3):
        for a, b in zip((tokens, q, p, u), inputs(dev, 6, 3, 5000, "fp32", seed)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, lm_head.verify_drafts(tokens, q, p, u)))


@pytest.mark.gpu
def test_compiled(dev):
    args = inputs(dev, 4, 2, 700, "bf16", 3)
    want = lm_head.verify_drafts(*args)
    got = torch.compile(lm_head.verify_drafts, fullgraph=True, backend="aot_eager")(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.library.opcheck(torch.ops.cinnamon_amd.verify_drafts.default, (*args, None))


def test_shapes_and_refusals():
    with FakeTensorMode():
        def t(*shape, dtype=torch.float32, device="cuda"):
            return torch.empty(*shape, dtype=dtype, device=device)

        i = torch.int64
        tokens, q, p, u = t(3, 2, dtype=i), t(3, 2, 50), t(3, 3, 50), t(3, 3)
        good = (tokens, q, p, u, t(3, dtype=torch.int32))
        for args in [(t(3, 2), q, p, u), (t(3, 2, dtype=torch.bool), q, p, u), (t(6, dtype=i), q, p, u), (tokens, q, t(3, 2, 50), u),
                     (tokens, t(3, 3, 50), p, u), (tokens, t(3, 2, 50, dtype=torch.bfloat16), p, u),
                     (tokens, q.double(), p.double(), u), (tokens, q, p, t(3, 2)), (tokens, q, p, t(3, 3, dtype=torch.float16)),
                     (tokens, q, p, u, t(2, dtype=i)), (tokens, q, p, u, t(3)), (t(3, 2, dtype=i, device="cpu"), q, p, u),
                     (tokens, q, t(3, 3, 50, device="cpu"), u), (tokens, t(3, 2, 0), t(3, 3, 0), u),
                     (t(1, 64, dtype=i), t(1, 64, 5), t(1, 65, 5), t(1, 65))]:
            with pytest.raises(AssertionError):
                lm_head.verify_drafts(*args)
        out, n = torch.ops.cinnamon_amd.verify_drafts(*good)
        assert out.shape == (3, 3) and n.shape == (3,) and out.dtype == n.dtype == i


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    big = 1 << 20

    def call(dtype=1, B=2, K=2, V=100, p=big, u=big, out=big, tokens=big, ws=(big, 1 << 20)):
        return lib.cin_verify_drafts(tokens, 2, 1, big, 200, 100, p, 300, 100, dtype, B, K, V, u, 0, 3, 1, None, 0, out, big, *ws, None)

    for kw in [dict(dtype=4), dict(B=-1), dict(B=65537), dict(K=64), dict(K=-1), dict(V=0), dict(V=1 << 30), dict(p=None), dict(u=None),
               dict(out=None), dict(tokens=None), dict(ws=(None, 0)), dict(ws=(big, 8)), dict(ws=(big + 8, 1 << 20)),
               dict(B=65536, V=(1 << 30) - 1)]:
        assert call(**kw) == _lib.CIN_ERR_ARG, kw
        assert _lib.last_error()
    assert call(B=0) == 0
    assert lib.cin_verify_drafts_workspace(1, 64, 100) == -1 and lib.cin_verify_drafts_workspace(0, 1, 100) == 0
