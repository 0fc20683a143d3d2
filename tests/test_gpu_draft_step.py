"""The norms around a block, the layer of a few tokens and the drafts' verification as a program uses them: together in a
generation step with drafted tokens and in a training step, next to the operators that were there."""
import math
import threading

import pytest
import torch
import torch.nn as nn

from cinnamon_amd import kernels, layers, lm_head, moe, norm


class Model(nn.Module):
    """Two blocks of norm, mixed experts, post norm and gated residual sum, and the output head; one draft head that
    shares it.  plain: the same in elementary operations on 64 bits."""

    def __init__(self, V=3000, D=256, H=128, E=8, k=2, blocks=2):
        super().__init__()
        g = torch.Generator().manual_seed(0)

        def p(*shape, std=1.0, mean=0.0):
            return nn.Parameter(torch.randn(*shape, generator=g) * std + mean)

        self.k = k
        self.emb = p(V, D)
        self.pre = nn.ParameterList([p(D, std=0.1, mean=1.0) for _ in range(blocks + 1)])
        self.post = nn.ParameterList([p(D, std=0.1, mean=1.0) for _ in range(blocks)])
        self.gate = nn.ParameterList([p(D, std=0.1, mean=0.5) for _ in range(blocks)])
        self.scale = nn.ParameterList([p(1, std=0.1, mean=0.9) for _ in range(blocks)])
        self.router = nn.ParameterList([p(E, D, std=0.1) for _ in range(blocks)])
        self.experts = nn.ModuleList([layers.GroupedExperts(E, D, H) for _ in range(blocks)])
        self.out = p(V, D, std=3 / math.sqrt(D))
        self.draft = p(D, D, std=1 / math.sqrt(D))
        with torch.no_grad():
            for e in self.experts:
                e.w12.copy_(torch.randn(e.w12.shape, generator=g) / math.sqrt(D))
                e.w3.copy_(torch.randn(e.w3.shape, generator=g) / math.sqrt(H))
        kernels.set_weight_cache(self)

    def step(self, ids):
        """Hidden states [n, D] of tokens after the last norm."""
        x = self.emb[ids].bfloat16()
        h = norm.rms_norm(x, self.pre[0])
        for i, e in enumerate(self.experts):
            y = moe.moe_decode(h, self.router[i], e, self.k)
            h, x = norm.block_norm(y, x, self.pre[i + 1], post_weight=self.post[i], gate=self.gate[i], residual_scale=self.scale[i])
        return h

    def plain(self, ids, chosen=None):
        def rms(v, w):
            return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()

        x = self.emb[ids].bfloat16().double()
        h = rms(x, self.pre[0])
        for i, e in enumerate(self.experts):
            s = torch.sigmoid(h @ self.router[i].double().t())
            w, idx = s.topk(self.k)
            w = w / (w.sum(-1, keepdim=True) + 1e-9)
            (q12, _, s12), (q3, _, s3) = layers.quantize_expert_weights(e.w12.detach(), e.w3.detach())
            E, H2, D = e.w12.shape
            wide = lambda q, s: q.double() * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)  # noqa: E731
            w12, w3 = wide(q12, s12).view(E, H2, D), wide(q3, s3).view(E, D, H2 // 2)
            y = torch.zeros_like(x)
            for j in range(self.k):
                a, b = (h[:, None] @ w12[idx[:, j]].transpose(1, 2))[:, 0].chunk(2, -1)
                y += w[:, j:j + 1] * ((torch.nn.functional.silu(a) * b)[:, None] @ w3[idx[:, j]].transpose(1, 2))[:, 0]
            x = self.scale[i].double() * x + self.gate[i].double() * rms(y, self.post[i])
            h = rms(x, self.pre[i + 1])
        return h


def probabilities(h, out):
    return torch.softmax(h.float() @ out.t(), -1)


@pytest.fixture(scope="module")
def model(dev):
    return Model().to(dev).requires_grad_(False)


def speculate(m, ids, K, u_draft, u):
    """K tokens drafted one behind the other by the draft head, then the target's step on all of them at once."""
    B = ids.shape[0]
    none = torch.empty(B, 0, dtype=torch.int64, device=ids.device)
    h = m.step(ids)
    tokens, q = [], []
    for i in range(K):
        p = probabilities(h.float() @ m.draft, m.out)
        # (a draw is the verification of no drafts)
        t = lm_head.verify_drafts(none, None, p[:, None], u_draft[:, i:i + 1])[0][:, 0]
        tokens.append(t)
        q.append(p)
        h = m.step(t)
    tokens, q = torch.stack(tokens, 1), torch.stack(q, 1)
    p = probabilities(m.step(torch.cat([ids[:, None], tokens], 1).flatten()), m.out).view(B, K + 1, -1)
    return (*lm_head.verify_drafts(tokens, q, p, u), tokens, q, p)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 40])
def test_hidden_states_of_a_step(dev, model, n):
    ids = torch.randint(0, 3000, (n,), generator=torch.Generator().manual_seed(1)).to(dev)
    h, want = model.step(ids), model.plain(ids)
    # bf16 roundings of h, y and x in each of two blocks, 2^-9 of a value at most and a third of its square on average; a
    # token whose second and third expert are as close as those roundings may choose the other: left out
    err = (h.double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert err.median() < 8 * 2.0 ** -9
    assert (err < 16 * 2.0 ** -9).double().mean() >= 0.9


@pytest.mark.gpu
def test_a_speculative_step(dev, model):
    B, K = 5, 3
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 3000, (B,), generator=g).to(dev)
    ud, u = torch.rand(B, K, generator=g).to(dev), torch.rand(B, K + 1, generator=g).to(dev)
    out, n, tokens, q, p = speculate(model, ids, K, ud, u)
    for b in range(B):
        for i in range(int(n[b])):
            assert out[b, i] == tokens[b, i]
            assert u[b, i].double() * q[b, i, tokens[b, i]].double() < p[b, i, tokens[b, i]].double()
        i = int(n[b])
        if i < K:
            assert u[b, i].double() * q[b, i, tokens[b, i]].double() >= p[b, i, tokens[b, i]].double()
            assert p[b, i, out[b, i]] > q[b, i, out[b, i]]
        assert (out[b, i + 1:] == -1).all() and 0 <= out[b, i] < 3000
    # drafts as likely as the target's own are all kept
    own = speculate(model, ids, 1, ud[:, :1], u[:, :2])
    same = lm_head.verify_drafts(own[2], own[4][:, :1], own[4], u[:, :2])
    assert (same[1] == 1).all()


@pytest.mark.gpu
def test_a_captured_step_replays(dev, model):
    B, K = 3, 2
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 3000, (B,), generator=g).to(dev)
    ud, u = torch.rand(B, K, generator=g).to(dev), torch.rand(B, K + 1, generator=g).to(dev)
    speculate(model, ids, K, ud, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        speculate(model, ids, K, ud, u)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = speculate(model, ids, K, ud, u)
    with torch.cuda.graph(other):
        held2 = speculate(model, ids, K, ud, u)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(0, 3000, (B,), generator=g))
        ud.copy_(torch.rand(B, K, generator=g))
        u.copy_(torch.rand(B, K + 1, generator=g))
        torch.cuda.synchronize()
        # both at once: neither has workspaces of the other's
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other.replay()
        graph.replay()
        torch.cuda.synchronize()
        want = speculate(model, ids, K, ud, u)
        for a, b, c in zip(held, held2, want):
            assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.gpu
def test_threads(dev, model):
    ids = torch.randint(0, 3000, (4, 6), generator=torch.Generator().manual_seed(4)).to(dev)
    want = [model.step(i) for i in ids]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = model.step(ids[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_training_step(dev):
    """Norms around an FP8 linear layer and the vocabulary loss: gradients against the same layers with the norms in
    elementary operations in 32 bits."""
    torch.manual_seed(5)
    D, V, T = 256, 1000, 96
    lin = kernels.FP8Linear(D, D).to(dev)
    with torch.no_grad():
        lin.weight.normal_(std=1 / 16)
    w, pw, g = (torch.randn(D, device=dev) * 0.1 + 1 for _ in range(3))
    a, out = torch.full((1,), 0.9, device=dev), torch.randn(V, D, device=dev) * 0.2
    x = torch.randn(T, D, device=dev)
    target = torch.randint(0, V, (T,), device=dev)
    leaves = [t.requires_grad_() for t in (x, w, pw, g, a, out)]

    def rms(v, w):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6) * w

    def loss(plain):
        h = rms(x, w) if plain else norm.rms_norm(x, w)
        y = lin(h).float()
        if plain:
            r = a * x + g * rms(y, pw)
            n = rms(r, w)
        else:
            n, r = norm.block_norm(y, x, w, post_weight=pw, gate=g, residual_scale=a)
        return lm_head.linear_cross_entropy(n, out, target) + r.square().mean()

    got, want = (torch.autograd.grad(loss(p), [*leaves, lin.weight]) for p in (False, True))
    for u, v in zip(got, want):
        # two fp32 forms of the norms; a code of the FP8 layer's input next to a border may round the other way, by 2^-4 of
        # one in some thousand values (2^-4 / sqrt(1000) of the norm)
        assert (u - v).norm() <= 2.0 ** -9 * v.norm()
