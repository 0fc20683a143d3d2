"""What is measured of the operators of a generation step with drafted tokens, and of the norms around
a block that training shares with it.

Kinds of case:
  norm    norm.block_norm: a block's output normed, gated and added to the scaled residual stream, and the
          next block's norm of the sum; where "train" also the gradients of all inputs
  moe     moe.moe_decode: a whole mixture-of-experts layer for a few tokens
  verify  lm_head.verify_drafts: drafted tokens against the target's probabilities
"""
import math

import numpy as np
import torch

own = False

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
_DT = {"bf16": BF16, "fp16": F16, "fp32": F32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
EPS = 1e-6


def listed():
    return [
        # a generation step of one sequence through the wide model: launches count
        {"name": "norm_token", "kind": "norm", "T": 1, "D": 7168, "x": "bf16", "r": "bf16", "w": "fp32", "post": False,
         "gate": "none", "scale": "one", "train": False},
        # the small training model, 16 x 1024 tokens, bf16 blocks on a residual stream in 32 bits
        {"name": "norm_train", "kind": "norm", "T": 16384, "D": 1024, "x": "bf16", "r": "fp32", "w": "fp32", "post": False,
         "gate": "none", "scale": "one", "train": True},
        # norms on both sides of the block, a gate per channel and a learned residual scale; the widest model
        {"name": "norm_train_large", "kind": "norm", "T": 16384, "D": 7168, "x": "bf16", "r": "bf16", "w": "fp32", "post": True,
         "gate": "channel", "scale": "scalar", "train": True},
        # a width that no vector divides, a gate per element from a modulation, a prompt's ragged length
        {"name": "norm_train_odd", "kind": "norm", "T": 4999, "D": 1111, "x": "fp16", "r": "fp16", "w": "fp16", "post": True,
         "gate": "element", "scale": "channel", "train": True},
        # one token of the small model: 16 experts, top-2, a shared expert of four times their width
        {"name": "moe_token_small", "kind": "moe", "T": 1, "D": 1024, "H": 1024, "E": 16, "k": 2, "shared": 4096, "x": "bf16",
         "wt": "fp8", "router": "fp32", "score": "sigmoid", "bias": True, "groups": 1, "top_groups": 1},
        # one token of the large routed layer: 32 experts, top-8
        {"name": "moe_token", "kind": "moe", "T": 1, "D": 7168, "H": 2048, "E": 32, "k": 8, "shared": 2048, "x": "bf16",
         "wt": "fp8", "router": "fp32", "score": "sigmoid", "bias": True, "groups": 1, "top_groups": 1},
        # a generation step of 64 sequences through it, experts in groups: the largest call
        {"name": "moe_batch", "kind": "moe", "T": 64, "D": 7168, "H": 2048, "E": 32, "k": 8, "shared": 2048, "x": "bf16",
         "wt": "fp8", "router": "fp32", "score": "sigmoid", "bias": True, "groups": 4, "top_groups": 3},
        # a few sequences through many small experts in 16 bits, widths that no block of 128 divides, fp32 states
        {"name": "moe_ragged", "kind": "moe", "T": 19, "D": 2000, "H": 720, "E": 60, "k": 4, "shared": 0, "x": "fp32",
         "wt": "bf16", "router": "bf16", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1},
        # one sequence with one draft head's token: latency
        {"name": "verify_one", "kind": "verify", "B": 1, "K": 1, "V": 32000, "p": "fp32", "ragged": False},
        # 64 sequences with four drafted tokens each, a large vocabulary
        {"name": "verify_batch", "kind": "verify", "B": 64, "K": 4, "V": 131072, "p": "fp32", "ragged": False},
        # sequences with different numbers of drafts, a vocabulary that nothing divides, 16-bit probabilities
        {"name": "verify_ragged", "kind": "verify", "B": 17, "K": 7, "V": 50257, "p": "bf16", "ragged": True},
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_norm(rng):
    step = rng.choice([128, 128, 8, 1])
    D = max(step, _log(rng, 64, 16384) // step * step)
    x = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    T = max(1, min(_log(rng, 1, 65536), 16384 * 7168 // (D * (2 if x == "fp32" else 1) * 2)))
    return {"kind": "norm", "T": T, "D": D, "x": x, "r": rng.choice([x, x, "fp32"]), "w": rng.choice(["fp32", x]),
            "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "token", "element"]),
            "scale": rng.choice(["one", "number", "scalar", "channel"]), "train": rng.random() < 0.7}


def _draw_moe(rng):
    wt = rng.choice(["fp8", "fp8", "bf16"])
    step = rng.choice([128, 128, 16])
    D = max(step, _log(rng, 256, 7168) // step * step)
    H = max(step, _log(rng, 128, 2048) // step * step)
    groups = rng.choice([1, 1, 2, 4, 8])
    most = 32 * 7168 * 2048 // (D * H) // (2 if wt == "bf16" else 1)
    E = groups * max(2, min(_log(rng, 8, 256), most) // groups)
    top_groups = rng.randint(1, groups)
    return {"kind": "moe", "T": rng.choice([1, _log(rng, 2, 64)]), "D": D, "H": H, "E": E,
            "k": rng.randint(1, min(8, top_groups * (E // groups))), "shared": rng.choice([0, H, 2 * H]),
            "x": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "wt": wt, "router": rng.choice(["fp32", "bf16"]),
            "score": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups}


def _draw_verify(rng):
    V = _log(rng, 1000, 131072)
    K = rng.randint(1, 8)
    B = max(1, min(_log(rng, 1, 128), 64 * 4 * 131072 // (K * V)))
    return {"kind": "verify", "B": B, "K": K, "V": V, "p": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
            "ragged": rng.random() < 0.5}


def draw(rng):
    return rng.choice([_draw_norm, _draw_moe, _draw_verify])(rng)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0, mean=0.0, dtype=F32):
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)


def _norm_inputs(c, seed):
    """A block's output (smaller than the stream, unless it is normed), the stream, the norms' weights
    around one, gates around a tenth and the gradients of both outputs."""
    g = _generator(seed)
    T, D, dt, wd = c["T"], c["D"], _DT[c["x"]], _DT[c["w"]]
    shape = {"channel": (D,), "token": (T, 1), "element": (T, D)}.get(c["gate"])
    s = {"y": _normal(g, T, D, std=0.4, dtype=dt), "residual": _normal(g, T, D, std=2.0, dtype=_DT[c["r"]]),
         "weight": _normal(g, D, std=0.2, mean=1.0, dtype=wd)}
    s["post_weight"] = _normal(g, D, std=0.2, mean=1.0, dtype=wd) if c["post"] else None
    s["gate"] = None if shape is None else _normal(g, *shape, std=0.1, mean=0.1, dtype=wd if c["gate"] == "channel" else dt)
    scale = c["scale"]
    s["residual_scale"] = {"one": lambda: None, "number": lambda: 0.875, "scalar": lambda: _normal(g, 1, std=0.1, mean=0.9),
                           "channel": lambda: _normal(g, D, std=0.1, mean=0.9, dtype=wd)}[scale]()
    s["gn"] = _normal(g, T, D, std=1e-2, dtype=dt) if c["train"] else None
    s["gr"] = _normal(g, T, D, std=1e-2, dtype=_DT[c["r"]]) if c["train"] else None
    return s


_NORM_LEAVES = ("y", "residual", "weight", "post_weight", "gate", "residual_scale")


def _blocks(w):
    """Codes and scales of the 128 x 128 blocks of w [R, C]: the largest value of a block becomes 448."""
    R, C = w.shape
    Rp, Cp = -(-R // 128), -(-C // 128)
    full = w.new_zeros(Rp * 128, Cp * 128)
    full[:R, :C] = w
    t = full.view(Rp, 128, Cp, 128)
    s = t.abs().amax(dim=(1, 3)).clamp_min(1e-4) / 448
    return (t / s[:, None, :, None]).view(Rp * 128, Cp * 128)[:R, :C].to(E4M3), s


def _weights(g, wt, rows, cols, std, E=None):
    """Weights [E, rows, cols] (or [rows, cols]) and their block scales; no scales in 16 bits."""
    if wt == "bf16":
        parts = [_normal(g, rows, cols, std=std, dtype=BF16) for _ in range(E or 1)]
        return (torch.stack(parts) if E else parts[0]), None
    parts = [_blocks(_normal(g, rows, cols, std=std)) for _ in range(E or 1)]
    if E is None:
        return parts[0]
    return torch.stack([q.view(torch.uint8) for q, _ in parts]).view(E4M3), torch.stack([s for _, s in parts])


def _moe_inputs(c, seed):
    """Hidden states after a norm, a router that likes some experts more, a balancing bias, and experts
    whose products keep the states' size."""
    g = _generator(seed)
    T, D, H, E, S = c["T"], c["D"], c["H"], c["E"], c["shared"]
    s = {"x": _normal(g, T, D, dtype=_DT[c["x"]]), "router": _normal(g, E, D, std=1.5 / math.sqrt(D), dtype=_DT[c["router"]]),
         "bias": _normal(g, E, std=0.05) if c["bias"] else None}
    w12, s12 = _weights(g, c["wt"], 2 * H, D, 1.5 / math.sqrt(D), E)
    w3, s3 = _weights(g, c["wt"], D, H, 1.5 / math.sqrt(H), E)
    s["experts"] = (w12, s12, w3, s3)
    s["shared"] = None
    if S:
        s["shared"] = (*_weights(g, c["wt"], 2 * S, D, 1.5 / math.sqrt(D)), *_weights(g, c["wt"], D, S, 1.5 / math.sqrt(S)))
    return s


def _verify_inputs(c, seed):
    """The target's probabilities as a softmax of peaked logits leaves them, those of draft heads that
    know them roughly, tokens drawn from the drafts' probabilities, and uniform numbers."""
    g = _generator(seed)
    B, K, V, dt = c["B"], c["K"], c["V"], _DT[c["p"]]
    z = _normal(g, B, K + 1, V, std=2.5)
    target = torch.softmax(z, -1)
    draft = torch.softmax(z[:, :K] + _normal(g, B, K, V, std=0.7), -1)
    pick = torch.rand(B * K, 1, device="cuda", generator=g, dtype=F64)
    cum = draft.view(B * K, V).double().cumsum(-1)
    tokens = torch.searchsorted(cum, pick * cum[:, -1:], right=True).clamp_max(V - 1).view(B, K)
    return {"tokens": tokens, "draft": draft.to(dt), "target": target.to(dt),
            "uniforms": torch.rand(B, K + 1, device="cuda", generator=g),
            "counts": torch.randint(0, K + 1, (B,), device="cuda", generator=g) if c["ragged"] else None}


_INPUTS = {"norm": _norm_inputs, "moe": _moe_inputs, "verify": _verify_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    if case["kind"] == "norm" and case["train"]:
        s["leaves"] = [s[n].requires_grad_() for n in _NORM_LEAVES if torch.is_tensor(s[n])]
    s["case"] = case
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _norm_plain(c, s):
    f = {n: v.detach().float() if torch.is_tensor(v) else v for n, v in s.items() if n in _NORM_LEAVES + ("gn", "gr")}
    y, r, w, pw, gate, a = (f[n] for n in _NORM_LEAVES)
    a = 1.0 if a is None else a
    u = y
    if c["post"]:
        inv_y = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        u = y * inv_y * pw
    x = a * r + (u if gate is None else gate * u)
    inv = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    out = {"normed": (x * inv * w).to(s["y"].dtype), "residual": x.to(s["residual"].dtype)}
    if not c["train"]:
        return out
    gn, gr = f["gn"], f["gr"]
    t = gn * w
    dx = gr + inv * (t - x * (inv * inv * (t * x).mean(-1, keepdim=True)))
    du = dx if gate is None else gate * dx
    dy = du
    if c["post"]:
        t = du * pw
        dy = inv_y * (t - y * (inv_y * inv_y * (t * y).mean(-1, keepdim=True)))
    g = {"y": dy, "residual": a * dx, "weight": (gn * x * inv).sum(0)}
    if c["post"]:
        g["post_weight"] = (du * y * inv_y).sum(0)
    if gate is not None:
        dg = dx * u
        g["gate"] = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(-1, keepdim=True), "element": lambda: dg}[c["gate"]]()
    if torch.is_tensor(a):
        da = dx * r
        g["residual_scale"] = da.sum().view(1) if c["scale"] == "scalar" else da.sum(0)
    out.update({"d_" + n: v.to(s[n].dtype) for n, v in g.items()})
    return out


def _largest(v, n):
    """Indices of the n largest of the last dimension, in falling order, ties to the lowest index."""
    return v.sort(dim=-1, descending=True, stable=True).indices[..., :n]


def _route_plain(c, x, router, bias):
    # in 64 bits: experts next to the border of the top k differ by less than 32 bits hold
    z = x.double() @ router.double().t()
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    choice = s if bias is None else s + bias.double()
    if c["groups"] > 1:
        T, G = z.shape[0], c["groups"]
        per = choice.view(T, G, -1)
        best = per.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter_(1, _largest(best, c["top_groups"]), True)
        choice = torch.where(kept[..., None], per, -math.inf).view(T, -1)
    idx = _largest(choice, c["k"])
    at = s.gather(1, idx)
    return idx, at / (at.sum(-1, keepdim=True) + 1e-9)


def _wide(w, scales):
    """Weights [.., R, C] in 32 bits."""
    if scales is None:
        return w.float()
    R, C = w.shape[-2:]
    s = scales.repeat_interleave(128, -2)[..., :R, :].repeat_interleave(128, -1)[..., :C]
    return w.float() * s


def _swiglu(x, w12, s12, w3, s3):
    h1, h2 = (x @ _wide(w12, s12).transpose(-1, -2)).chunk(2, dim=-1)
    return (h1 / (1 + torch.exp(-h1)) * h2) @ _wide(w3, s3).transpose(-1, -2)


def _moe_plain(c, s):
    T, E, k = c["T"], c["E"], c["k"]
    x = s["x"].float()
    idx, weights = _route_plain(c, s["x"], s["router"], s["bias"])
    wf = weights.float()
    w12, s12, w3, s3 = s["experts"]
    pick = lambda t, i: None if t is None else t.view(torch.uint8)[i].view(E4M3) if t.dtype == E4M3 else t[i]  # noqa: E731
    if T * k <= E:  # only the chosen experts' weights
        i = idx.reshape(-1)
        rows = x.repeat_interleave(k, 0)[:, None]
        y = _swiglu(rows, *(pick(t, i) for t in (w12, s12, w3, s3)))
        out = (y.view(T, k, -1) * wf[..., None]).sum(1)
    else:
        dense = torch.zeros(T, E, device=x.device).scatter_(1, idx, wf)
        out = torch.zeros_like(x)
        for e in range(E):
            out += _swiglu(x, *(pick(t, e) for t in (w12, s12, w3, s3))) * dense[:, e:e + 1]
    if s["shared"] is not None:
        out = out + _swiglu(x, *s["shared"])
    return {"out": out.to(s["x"].dtype), "idx": idx, "weights": wf}


def _verify_plain(c, s):
    # in 64 bits: a sum over the vocabulary decides on which side of a border a number falls
    B, K, V = c["B"], c["K"], c["V"]
    tokens, u = s["tokens"], s["uniforms"].double()
    p = s["target"][:, :K].gather(2, tokens[..., None])[..., 0].double()
    q = s["draft"].gather(2, tokens[..., None])[..., 0].double()
    ok = u[:, :K] * q < p
    if s["counts"] is not None:
        ok &= torch.arange(K, device=ok.device) < s["counts"][:, None]
    n = ok.long().cumprod(1).sum(1)
    limit = torch.full_like(n, K) if s["counts"] is None else s["counts"]
    b = torch.arange(B, device=n.device)
    row = s["target"][b, n].double()
    drafted = torch.where((n < limit)[:, None], s["draft"][b, n.clamp_max(K - 1)].double(), 0)
    rest = (row - drafted).clamp_min(0)
    rest = torch.where((rest.sum(-1, keepdim=True) > 0), rest, row)
    cum = rest.cumsum(-1)
    # the first entry whose sum passes the number's share of the whole
    new = (cum <= u[:, K:] * cum[:, -1:]).sum(-1).clamp_max(V - 1)
    at = torch.arange(K + 1, device=n.device)
    out = torch.where(at < n[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    return {"tokens": torch.where(at == n[:, None], new[:, None], out), "accepted": n}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _norm_own(c, s):
    from cinnamon_amd import norm
    n, r = norm.block_norm(s["y"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                           residual_scale=s["residual_scale"], eps=EPS)
    if not c["train"]:
        return {"normed": n, "residual": r}
    grads = torch.autograd.grad([n, r], s["leaves"], [s["gn"], s["gr"]])
    names = [m for m in _NORM_LEAVES if torch.is_tensor(s[m])]
    return {"normed": n.detach(), "residual": r.detach(), **{"d_" + m: v for m, v in zip(names, grads)}}


def _moe_own(c, s):
    from cinnamon_amd import moe
    out, idx, weights = moe.moe_decode(s["x"], s["router"], s["experts"], c["k"], bias=s["bias"], score=c["score"],
                                       n_groups=c["groups"], top_groups=c["top_groups"], shared=s["shared"],
                                       return_routing=True)
    return {"out": out, "idx": idx, "weights": weights}


def _verify_own(c, s):
    from cinnamon_amd import lm_head
    tokens, accepted = lm_head.verify_drafts(s["tokens"], s["draft"], s["target"], s["uniforms"], n_drafts=s["counts"])
    return {"tokens": tokens, "accepted": accepted}


_PLAIN = {"norm": _norm_plain, "moe": _moe_plain, "verify": _verify_plain}
_OWN = {"norm": _norm_own, "moe": _moe_own, "verify": _verify_own}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "norm":
        T, D, es, rs, ws = c["T"], c["D"], _ES[c["x"]], _ES[c["r"]], _ES[c["w"]]
        gate = {"none": 0, "channel": D * ws, "token": T * es, "element": T * D * es}[c["gate"]]
        scale = {"channel": D * ws, "scalar": 4}.get(c["scale"], 0)
        small = D * ws * (2 if c["post"] else 1) + gate + scale
        both = 2 if c["train"] else 1
        # forward: y and r in, both outputs out; backward: both outputs' gradients in, those of y and r out
        return {"bytes": both * (2 * T * D * (es + rs) + small), "flops": both * T * D * (12 if c["post"] else 7)}
    if c["kind"] == "moe":
        T, D, H, E, k, S = c["T"], c["D"], c["H"], c["E"], c["k"], c["shared"]
        per = _ES[c["wt"]] + (4 / 16384 if c["wt"] == "fp8" else 0)
        chosen = E * (1 - (1 - k / E) ** T)  # experts that are some token's, if all are liked alike
        b = 3 * D * (chosen * H + S) * per + E * D * _ES[c["router"]] + 2 * T * D * _ES[c["x"]] + 12 * T * k
        return {"bytes": int(b), "flops": 2 * T * D * (E + 3 * (k * H + S))}
    B, K, V = c["B"], c["K"], c["V"]
    # a row of each side's probabilities, and the drafts' own entries
    return {"bytes": B * (2 * V * _ES[c["p"]] + K * (2 * _ES[c["p"]] + 20)), "flops": 3 * B * V}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _norm_exact(c, seed):
    s = _norm_inputs(c, seed)
    leaf = {n: s[n].double().requires_grad_(c["train"]) for n in _NORM_LEAVES if torch.is_tensor(s[n])}
    rms = lambda v: v * (v.square().sum(-1, keepdim=True) / c["D"] + EPS).rsqrt()  # noqa: E731
    block = rms(leaf["y"]) * leaf["post_weight"] if c["post"] else leaf["y"]
    if "gate" in leaf:
        block = block * leaf["gate"]
    scale = leaf.get("residual_scale", s["residual_scale"])
    stream = leaf["residual"] if scale is None else leaf["residual"] * scale
    stream = stream + block
    normed = rms(stream) * leaf["weight"]
    r = {"normed": normed.detach(), "residual": stream.detach()}
    if c["train"]:
        ((normed * s["gn"].double()).sum() + (stream * s["gr"].double()).sum()).backward()
        r.update({"d_" + n: v.grad for n, v in leaf.items()})
    return r


def _moe_exact(c, seed):
    s = _moe_inputs(c, seed)
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    x = s["x"].double()
    z = (x.cpu().numpy()[:, None, :] * s["router"].double().cpu().numpy()[None]).sum(-1)
    if c["score"] == "sigmoid":
        score = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
    else:
        score = np.exp(z - z.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    choice = score + (0.0 if s["bias"] is None else s["bias"].double().cpu().numpy())
    rows = np.arange(T)[:, None]
    if G > 1:
        low = np.sort(choice.reshape(T, G, -1), axis=2)
        best = low[:, :, -2:].sum(-1)
        blocked = np.zeros((T, G), bool)
        blocked[rows, np.argsort(-best, axis=1, kind="stable")[:, c["top_groups"]:]] = True
        choice = np.where(np.repeat(blocked, E // G, axis=1), -np.inf, choice)
    idx = np.argsort(-choice, axis=1, kind="stable")[:, :k]
    at = score[rows, idx]
    weights = at / (at.sum(1, keepdims=True) + 1e-9)

    def values(w, scales):
        if scales is None:
            return w.double()
        R, C = w.shape
        i, j = torch.arange(R, device=w.device) // 128, torch.arange(C, device=w.device) // 128
        return w.float().double() * scales.double()[i][:, j]

    def expert(rows, w12, s12, w3, s3):
        a, b = (rows @ values(w12, s12).t()).tensor_split(2, dim=-1)
        return (a * torch.sigmoid(a) * b) @ values(w3, s3).t()

    out = torch.zeros_like(x)
    for e in np.unique(idx):
        t, j = np.nonzero(idx == e)
        t = torch.from_numpy(t).to(x.device)
        w = torch.from_numpy(weights[t.cpu().numpy(), j]).to(x.device)
        out[t] += expert(x[t], *(None if v is None else v[int(e)] for v in s["experts"])) * w[:, None]
    if s["shared"] is not None:
        out += expert(x, *s["shared"])
    return {"out": out, "idx": torch.from_numpy(idx).to(x.device), "weights": torch.from_numpy(weights).to(x.device)}


def _verify_exact(c, seed):
    s = _verify_inputs(c, seed)
    B, K = c["B"], c["K"]
    tokens, u = s["tokens"].cpu().numpy(), s["uniforms"].cpu().numpy().astype(np.float64)
    out, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        p = s["target"][b].double().cpu().numpy()
        q = s["draft"][b].double().cpu().numpy()
        limit = K if s["counts"] is None else int(s["counts"][b])
        n = 0
        while n < limit and u[b, n] * q[n, tokens[b, n]] < p[n, tokens[b, n]]:
            out[b, n] = tokens[b, n]
            n += 1
        rest = np.maximum(p[n] - q[n], 0) if n < limit else p[n]
        if not rest.any():
            rest = p[n]
        cum = np.cumsum(rest)
        out[b, n] = np.searchsorted(cum, u[b, K] * cum[-1], side="right")
        accepted[b] = n
    return {"tokens": torch.from_numpy(out).cuda(), "accepted": torch.from_numpy(accepted).cuda()}


def exact(case, seed):
    return {"norm": _norm_exact, "moe": _moe_exact, "verify": _verify_exact}[case["kind"]](case, seed)
