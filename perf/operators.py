"""What is measured of the operators around the FP8 layers of a training or serving step: the
experts' gate, the rotary positions and the loss over the vocabulary.

Kinds of case:
  gate    moe.moe_gate: expert scores, the chosen experts and their weights; where "train" also
          all scores (a balance loss reads them) and the gradient of the logits
  rotary  rotary.apply_rotary on queries and keys; where "train" also their gradients
  loss    lm_head.linear_cross_entropy; where "train" also the gradients of the hidden states
          and of the output weights
"""
import math

import numpy as np
import torch

own = False

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
_DT = {"bf16": BF16, "fp16": F16, "fp32": F32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a generation step of 64 sequences in the large routed layer: 32 experts, top-8; launches count
        {"name": "gate_decode", "kind": "gate", "T": 64, "E": 32, "k": 8, "score": "sigmoid", "bias": True, "groups": 1,
         "top_groups": 1, "group_top": 2, "x": "fp32", "train": False},
        # the router of the small training model, 16 x 1024 tokens, 16 experts, top-2
        {"name": "gate_train", "kind": "gate", "T": 16384, "E": 16, "k": 2, "score": "sigmoid", "bias": True, "groups": 1,
         "top_groups": 1, "group_top": 2, "x": "fp32", "train": True},
        # many experts in groups, as expert-parallel layers limit a token to some nodes; the largest router
        {"name": "gate_train_groups", "kind": "gate", "T": 65536, "E": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "x": "bf16", "train": True},
        # a ragged prompt through a softmax router whose groups count by their best expert, no bias
        {"name": "gate_prefill_softmax", "kind": "gate", "T": 4999, "E": 160, "k": 6, "score": "softmax", "bias": False,
         "groups": 8, "top_groups": 3, "group_top": 1, "x": "fp16", "train": False},
        # a generation step: 64 sequences, each at its own position, heads of 64 + 64 rotated channels
        {"name": "rotary_decode", "kind": "rotary", "B": 64, "L": 1, "H": 16, "Hk": 1, "D": 128, "start": 64, "rot": 64,
         "interleaved": True, "P": 32768, "scaled": False, "positions": "each", "x": "bf16", "train": False},
        # the rotated channels of the small training model, 16 x 1024 tokens, one key head
        {"name": "rotary_train", "kind": "rotary", "B": 16, "L": 1024, "H": 16, "Hk": 1, "D": 64, "start": 0, "rot": 64,
         "interleaved": True, "P": 1024, "scaled": False, "positions": "none", "x": "bf16", "train": True},
        # a long prompt's last part at far positions of a stretched context, half layout, part of a wide head
        {"name": "rotary_long", "kind": "rotary", "B": 1, "L": 32767, "H": 16, "Hk": 16, "D": 192, "start": 128, "rot": 64,
         "interleaved": False, "P": 131072, "scaled": True, "positions": "far", "x": "fp16", "train": False},
        # the likelihood of a few generated tokens: the output weights are read once
        {"name": "loss_score", "kind": "loss", "T": 16, "V": 32000, "D": 1024, "x": "bf16", "reduction": "none",
         "ignored": 0.0, "train": False},
        # the small training model's loss on 16 x 1023 rows
        {"name": "loss_train", "kind": "loss", "T": 16368, "V": 32000, "D": 1024, "x": "bf16", "reduction": "mean",
         "ignored": 0.0, "train": True},
        # the same model as it trains in fp32, a small batch
        {"name": "loss_train_fp32", "kind": "loss", "T": 2046, "V": 32000, "D": 1024, "x": "fp32", "reduction": "mean",
         "ignored": 0.0, "train": True},
        # chat tuning: prompts masked, a vocabulary and a width that no tile divides
        {"name": "loss_tune_odd", "kind": "loss", "T": 3001, "V": 50257, "D": 1001, "x": "fp16", "reduction": "sum",
         "ignored": 0.4, "train": True},
        # a large vocabulary and a wide model, the largest call
        {"name": "loss_train_large", "kind": "loss", "T": 8192, "V": 131072, "D": 4096, "x": "bf16", "reduction": "mean",
         "ignored": 0.05, "train": True},
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_gate(rng):
    groups = rng.choice([1, 1, 2, 4, 8])
    E = groups * _log(rng, 4, 64 if groups > 1 else 384)
    top_groups = rng.randint(1, groups)
    T = min(_log(rng, 1, 65536), 65536 * 256 // E)
    return {"kind": "gate", "T": T, "E": E, "k": rng.randint(1, min(10, top_groups * (E // groups))),
            "score": rng.choice(["sigmoid", "sigmoid", "softmax"]), "bias": rng.random() < 0.6, "groups": groups,
            "top_groups": top_groups, "group_top": rng.choice([1, 2]), "x": rng.choice(["bf16", "fp16", "fp32"]),
            "train": rng.random() < 0.6}


def _draw_rotary(rng):
    rot = rng.choice([16, 32, 64, 64, 128])
    start = rng.choice([0, 0, 16, 64, 128])
    D = start + rot + rng.choice([0, 0, 32, 1])
    H, Hk = rng.choice([1, 4, 12, 16, 32]), rng.choice([1, 1, 4, 8])
    B = _log(rng, 1, 64)
    L = 1 if rng.random() < 0.3 else max(1, min(_log(rng, 2, 32768), 32767 * 32 * 192 // (2 * B * (H + Hk) * D)))
    return {"kind": "rotary", "B": B, "L": L, "H": H, "Hk": Hk, "D": D, "start": start, "rot": rot,
            "interleaved": rng.random() < 0.5, "P": max(L, _log(rng, 1024, 131072)), "scaled": rng.random() < 0.4,
            "positions": rng.choice(["none", "far", "each"]), "x": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "train": rng.random() < 0.5}


def _draw_loss(rng):
    x = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    V = _log(rng, 1000, 131072)
    D = _log(rng, 128, 4096)
    step = rng.choice([64, 64, 64, 8, 1])
    D = max(step, D // step * step)
    most = 2046 * 32000 * 1024 * 4 if x == "fp32" else 8192 * 131072 * 4096 // 2
    T = max(1, min(_log(rng, 1, 16384), most // (V * D)))
    return {"kind": "loss", "T": T, "V": V, "D": D, "x": x, "reduction": rng.choice(["mean", "sum", "none"]),
            "ignored": rng.choice([0.0, 0.1, 0.5]), "train": rng.random() < 0.7}


def draw(rng):
    return rng.choice([_draw_gate, _draw_rotary, _draw_loss])(rng)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _gate_inputs(c, seed):
    """Logits of a router with popular and unpopular experts, a balancing bias about as large as
    the scores' spread, and gradients of the weights and of all scores."""
    g = _generator(seed)
    popular = _normal(g, c["E"], std=0.7)
    logits = (_normal(g, c["T"], c["E"]) + popular).to(_DT[c["x"]])
    bias = _normal(g, c["E"], std=0.05) if c["bias"] else None
    gw = _normal(g, c["T"], c["k"], std=1e-2) if c["train"] else None
    gs = _normal(g, c["T"], c["E"], std=1e-4) if c["train"] else None
    return logits, bias, gw, gs


def _tables(c):
    """cos and sin [P, rot / 2] of position times frequency, taken in 64 bits; "scaled" divides the
    slow frequencies by 8 and leaves the fast ones, with a ramp between, and scales both tables by
    the attention factor of that stretch."""
    n = c["rot"] // 2
    freq = 10000.0 ** (-torch.arange(n, device="cuda", dtype=F64) / n)
    factor = 1.0
    if c["scaled"]:
        turns = c["P"] / 8 * freq / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freq = freq * keep + freq / 8 * (1 - keep)
        factor = 0.1 * math.log(8) + 1
    angle = torch.arange(c["P"], device="cuda", dtype=F64)[:, None] * freq
    return (angle.cos() * factor).to(F32), (angle.sin() * factor).to(F32)


def _rotary_inputs(c, seed):
    g = _generator(seed)
    B, L, D, P = c["B"], c["L"], c["D"], c["P"]
    dt = _DT[c["x"]]
    q, k = _normal(g, B, L, c["H"], D, dtype=dt), _normal(g, B, L, c["Hk"], D, dtype=dt)
    gq = _normal(g, B, L, c["H"], D, std=1e-2, dtype=dt) if c["train"] else None
    gk = _normal(g, B, L, c["Hk"], D, std=1e-2, dtype=dt) if c["train"] else None
    along = torch.arange(L, device="cuda")
    if c["positions"] == "none":
        positions = None
    elif c["positions"] == "far":
        positions = along + (P - L)
    else:
        positions = along + torch.randint(0, P - L + 1, (B, 1), device="cuda", generator=g)
    return q, k, gq, gk, positions


def _loss_inputs(c, seed):
    """Hidden states after a norm and output weights that give logits a spread of about 2, with the
    targets' logits raised as training raises them (by up to 8, some still low)."""
    g = _generator(seed)
    T, V, D, dt = c["T"], c["V"], c["D"], _DT[c["x"]]
    w = _normal(g, V, D, std=2 / math.sqrt(D))
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    lift = torch.rand(T, 1, device="cuda", generator=g) * 2
    x = (_normal(g, T, D) + lift * w[target]).to(dt)
    target = torch.where(torch.rand(T, device="cuda", generator=g) < c["ignored"], -100, target)
    gr = _normal(g, T, std=1.0) if c["train"] and c["reduction"] == "none" else None
    return x, w.to(dt), target, gr


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "gate":
        s["logits"], s["bias"], s["gw"], s["gs"] = _gate_inputs(case, seed)
        s["logits"].requires_grad_(case["train"])
    elif case["kind"] == "rotary":
        s["q"], s["k"], s["gq"], s["gk"], s["positions"] = _rotary_inputs(case, seed)
        s["cos"], s["sin"] = _tables(case)  # kept by a program beside its weights
        s["q"].requires_grad_(case["train"])
        s["k"].requires_grad_(case["train"])
    else:
        s["x"], s["w"], s["target"], s["gr"] = _loss_inputs(case, seed)
        s["x"].requires_grad_(case["train"])
        s["w"].requires_grad_(case["train"])
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _largest(v, n):
    """Indices of the n largest of the last dimension, in falling order, ties to the lowest index."""
    return v.sort(dim=-1, descending=True, stable=True).indices[..., :n]


def _gate_plain(c, logits, bias, gw, gs):
    # scores in 64 bits: experts next to the border of the top k differ by less than 32 bits hold
    z = logits.detach().double()
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    choice = s if bias is None else s + bias.double()
    if c["groups"] > 1:
        T, G, n = c["T"], c["groups"], c["E"] // c["groups"]
        per = choice.view(T, G, n)
        best = per.sort(dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        kept = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter_(1, _largest(best, c["top_groups"]), True)
        choice = torch.where(kept[..., None], per, -math.inf).view(T, -1)
    idx = _largest(choice, c["k"])
    at = s.gather(1, idx)
    total = at.sum(-1, keepdim=True) + 1e-9
    w = at / total
    if not c["train"]:
        return {"idx": idx, "weights": w.float()}
    gwd = gw.double()
    ds = gs.double().scatter_add(1, idx, (gwd - (gwd * w).sum(-1, keepdim=True)) / total)
    if c["score"] == "sigmoid":
        dz = ds * s * (1 - s)
    else:
        dz = s * (ds - (ds * s).sum(-1, keepdim=True))
    return {"idx": idx, "weights": w.float(), "scores": s.float(), "dlogits": dz.to(logits.dtype)}


def _rotate_plain(c, x, cos, sin):
    """x with the pairs of its rotated channels turned by the angles of cos and sin [.., 1, rot / 2]."""
    a, r = c["start"], c["rot"]
    xf = x.detach().float()
    part = xf[..., a:a + r]
    if c["interleaved"]:
        x0, x1 = part[..., 0::2], part[..., 1::2]
    else:
        x0, x1 = part[..., :r // 2], part[..., r // 2:]
    y0, y1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    turned = torch.stack([y0, y1], -1).flatten(-2) if c["interleaved"] else torch.cat([y0, y1], -1)
    return torch.cat([xf[..., :a], turned, xf[..., a + r:]], -1).to(x.dtype)


def _rotary_plain(c, s):
    at = torch.arange(c["L"], device="cuda") if s["positions"] is None else s["positions"]
    cos, sin = s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2)
    out = {"q": _rotate_plain(c, s["q"], cos, sin), "k": _rotate_plain(c, s["k"], cos, sin)}
    if c["train"]:
        out["dq"], out["dk"] = _rotate_plain(c, s["gq"], cos, -sin), _rotate_plain(c, s["gk"], cos, -sin)
    return out


def _loss_plain(c, x, w, target, gr):
    xf, wf = x.detach().float(), w.detach().float()
    z = xf @ wf.t()
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - m)
    total = p.sum(-1, keepdim=True)
    kept = target != -100
    at = torch.where(kept, target, 0)[:, None]
    rows = torch.where(kept, (m + total.log() - z.gather(1, at))[:, 0], 0)
    n = kept.sum().float()
    loss = {"none": lambda: rows, "sum": rows.sum, "mean": lambda: rows.sum() / n}[c["reduction"]]()
    if not c["train"]:
        return {"loss": loss}
    g = kept.float() / n if c["reduction"] == "mean" else kept.float() if gr is None else kept * gr
    del z
    dz = p.div_(total).scatter_add_(1, at, torch.full_like(rows, -1.0)[:, None]).mul_(g[:, None])
    return {"loss": loss, "dx": (dz @ wf).to(x.dtype), "dw": (dz.t() @ xf).to(w.dtype)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _gate_own(c, logits, bias, gw, gs):
    from cinnamon_amd import moe
    r = moe.moe_gate(logits, c["k"], bias=bias, score=c["score"], n_groups=c["groups"], top_groups=c["top_groups"],
                     group_top=c["group_top"], return_scores=c["train"])
    if not c["train"]:
        return {"idx": r[0], "weights": r[1]}
    (dlogits,) = torch.autograd.grad([r[1], r[2]], [logits], [gw, gs])
    return {"idx": r[0], "weights": r[1].detach(), "scores": r[2].detach(), "dlogits": dlogits}


def _rotary_own(c, s):
    from cinnamon_amd import rotary
    q, k = rotary.apply_rotary(s["q"], s["cos"], s["sin"], k=s["k"], positions=s["positions"],
                               interleaved=c["interleaved"], start=c["start"])
    if not c["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["gq"], s["gk"]])
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _loss_own(c, x, w, target, gr):
    from cinnamon_amd import lm_head
    loss = lm_head.linear_cross_entropy(x, w, target, reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [x, w], gr)
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def run(state):
    c = state["case"]
    if c["kind"] == "gate":
        return (_gate_own if own else _gate_plain)(c, state["logits"], state["bias"], state["gw"], state["gs"])
    if c["kind"] == "rotary":
        return (_rotary_own if own else _rotary_plain)(c, state)
    return (_loss_own if own else _loss_plain)(c, state["x"], state["w"], state["target"], state["gr"])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, es = case, _ES[case["x"]]
    if c["kind"] == "gate":
        T, E, k = c["T"], c["E"], c["k"]
        b = T * E * es + 4 * E * c["bias"] + 12 * T * k
        if c["train"]:
            b += 4 * T * E + 4 * T * k + 4 * T * E + T * E * es  # scores out, their and the weights' gradients in, dlogits
        return {"bytes": b, "flops": T * E * (16 if c["train"] else 8)}
    if c["kind"] == "rotary":
        n = c["B"] * c["L"] * (c["H"] + c["Hk"])
        rows = c["B"] * c["L"] if c["positions"] == "each" else c["L"]
        both = 2 if c["train"] else 1
        b = both * 2 * n * c["D"] * es + min(rows, c["P"]) * c["rot"] * 4 + (0 if c["positions"] == "none" else 8 * rows)
        return {"bytes": b, "flops": both * 3 * n * c["rot"]}
    T, V, D = c["T"], c["V"], c["D"]
    b = (T + V) * D * es + 8 * T + (4 * T if c["reduction"] == "none" else 4)
    if not c["train"]:
        return {"bytes": b, "flops": 2 * T * V * D}
    return {"bytes": b + (T + V) * D * es + (4 * T if c["reduction"] == "none" else 0), "flops": 6 * T * V * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _gate_exact(c, seed):
    logits, bias, gw, gs = _gate_inputs(c, seed)
    dev = logits.device
    z = logits.float().cpu().numpy().astype(np.float64)
    T, E = z.shape
    G, n, rows = c["groups"], E // c["groups"], np.arange(T)[:, None]
    if c["score"] == "sigmoid":
        s = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
    else:
        s = np.exp(z - z.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
    choice = s + (0.0 if bias is None else bias.cpu().numpy().astype(np.float64))
    if G > 1:
        low = np.sort(choice.reshape(T, G, n), axis=2)
        best = low[:, :, -1] + (low[:, :, -2] if c["group_top"] == 2 and n > 1 else 0.0)
        out = np.argsort(-best, axis=1, kind="stable")[:, c["top_groups"]:]
        blocked = np.zeros((T, G), bool)
        blocked[rows, out] = True
        choice = np.where(np.repeat(blocked, n, axis=1), -np.inf, choice)
    idx = np.argsort(-choice, axis=1, kind="stable")[:, :c["k"]]
    at = s[rows, idx]
    total = at.sum(1, keepdims=True) + 1e-9
    r = {"idx": torch.from_numpy(idx).to(dev), "weights": torch.from_numpy(at / total).to(dev)}
    if c["train"]:
        gwd, ds = gw.cpu().numpy().astype(np.float64), gs.cpu().numpy().astype(np.float64)
        # w_j = s_j / total: dw_j / ds_i = [i = j] / total - s_j / total^2
        ds[rows, idx] += gwd / total - (gwd * at).sum(1, keepdims=True) / total ** 2
        dz = ds * s * (1 - s) if c["score"] == "sigmoid" else s * ds - s * (s * ds).sum(1, keepdims=True)
        r["scores"], r["dlogits"] = torch.from_numpy(s).to(dev), torch.from_numpy(dz).to(dev)
    return r


def _rotary_exact(c, seed):
    q, k, gq, gk, positions = _rotary_inputs(c, seed)
    cos, sin = _tables(c)
    at = torch.arange(c["L"], device="cuda") if positions is None else positions
    turn = torch.complex(cos[at].double(), sin[at].double()).unsqueeze(-2)
    a, r = c["start"], c["rot"]

    def rotate(x, by):
        y = x.double()
        if c["interleaved"]:
            v = torch.view_as_complex(y[..., a:a + r].reshape(*y.shape[:-1], r // 2, 2).contiguous()) * by
            y[..., a:a + r] = torch.view_as_real(v).flatten(-2)
        else:
            v = torch.complex(y[..., a:a + r // 2].contiguous(), y[..., a + r // 2:a + r].contiguous()) * by
            y[..., a:a + r // 2], y[..., a + r // 2:a + r] = v.real, v.imag
        return y

    out = {"q": rotate(q, turn), "k": rotate(k, turn)}
    if c["train"]:
        out["dq"], out["dk"] = rotate(gq, turn.conj()), rotate(gk, turn.conj())
    return out


def _loss_exact(c, seed):
    """By pieces of the vocabulary, so that the logits in 64 bits fit beside the rest."""
    x, w, target, gr = _loss_inputs(c, seed)
    T, V = c["T"], c["V"]
    xd, kept = x.double(), target >= 0
    step = max(1, min(V, (1 << 28) // T))
    m = torch.full((T,), -math.inf, dtype=F64, device="cuda")
    total, zt = torch.zeros_like(m), torch.zeros_like(m)
    for v in range(0, V, step):
        z = xd @ w[v:v + step].double().t()
        new = torch.maximum(m, z.amax(1))
        total = total * torch.exp(m - new) + torch.exp(z - new[:, None]).sum(1)
        m = new
        here = kept & (target >= v) & (target < v + step)
        zt[here] = z[here, target[here] - v]
    lse = m + total.log()
    rows = torch.where(kept, lse - zt, 0.0)
    n = kept.sum()
    loss = rows if c["reduction"] == "none" else rows.sum() / (n if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return {"loss": loss}
    g = kept.double() / n if c["reduction"] == "mean" else kept.double() * (1.0 if gr is None else gr.double())
    dx, dw = torch.zeros_like(xd), torch.empty(V, c["D"], dtype=F64, device="cuda")
    for v in range(0, V, step):
        wd = w[v:v + step].double()
        dz = torch.exp(xd @ wd.t() - lse[:, None])
        here = (kept & (target >= v) & (target < v + step)).nonzero()[:, 0]
        dz[here, target[here] - v] -= 1
        dz *= g[:, None]
        dx += dz @ wd
        dw[v:v + step] = dz.t() @ xd
    return {"loss": loss, "dx": dx, "dw": dw}


def exact(case, seed):
    return {"gate": _gate_exact, "rotary": _rotary_exact, "loss": _loss_exact}[case["kind"]](case, seed)
