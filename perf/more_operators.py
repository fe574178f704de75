"""The operators at the ends of a decoder of packed linear layers and in the seams between its
layers: the embedding with its gradient, the norms before and after a block with its gate and
residual, and the log probabilities of tokens under a large vocabulary without its logits being
kept, with the gradients of the hidden states and of the head.

``listed`` holds the cases that are timed and ``draw`` gives more of the same ranges.  With
``own`` false a pass computes the operator in plain fp32 torch operations, with it true it makes
the framework's calls; both work on the tensors that ``prepare`` makes.

    embed  out = scale W[token], 0 for a token outside the vocabulary; with a gradient also the
           dense gradient of W [vocab, width]
    norm   b = branch rsqrt(mean branch^2 + eps) branch_weight   (or the branch as it is)
           h = x + scale gate b
           y = h rsqrt(mean h^2 + eps) weight
    head   logprob = l[token] - log sum exp l and entropy = -sum p log p for l = hidden W^T; W in 16
           bits, or packed: E2M1 codes, two a byte, and an E8M0 scale for 32 of them
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
MOST_WEIGHTS = 131072 * 4096         # vocabulary x width of the largest listed head or embedding
MOST_PRODUCT = 4096 * MOST_WEIGHTS   # rows x vocabulary x width of the largest listed head
MOST_NORM = 8192 * 8192              # rows x width of the largest listed norm without a gradient
MOST_NORM_GRAD = 8192 * 4096         # and with one
MOST_EMBEDDED = 16384 * 2048         # tokens x width of the largest listed embedding


def _embed(name, rows, vocab, width, dt, grad, padded=0.0):
    return {"name": name, "kind": "embed", "rows": rows, "vocab": vocab, "width": width, "dt": dt,
            "grad": grad, "padded": padded}


def _norm(name, B, T, width, dt, wdt, gate, post, grad):
    return {"name": name, "kind": "norm", "B": B, "T": T, "width": width, "dt": dt, "wdt": wdt,
            "gate": gate, "post": post, "grad": grad}


def _head(name, rows, vocab, width, dt, packed, grad, entropy=False, padded=0.0):
    return {"name": name, "kind": "head", "rows": rows, "vocab": vocab, "width": width, "dt": dt,
            "packed": packed, "grad": grad, "entropy": entropy, "padded": padded}


def listed():
    return [
        # the next token of each of four sequences that are being answered
        _embed("embed_4x4096", 4, 32000, 4096, "bf16", False),
        # a training step's batch: the lookup and the gradient of a vocabulary of 32,000
        _embed("embed_train_4096x4096", 4096, 32000, 4096, "bf16", True),
        # a long batch with padding, a large vocabulary held in fp32
        _embed("embed_train_16384x2048_f32", 16384, 131072, 2048, "f32", True, 0.1),
        # one token while answering: the seam between two blocks
        _norm("norm_1x4096", 1, 1, 4096, "bf16", "f32", "none", False, False),
        # a long prompt through a wide model with norms on both sides of a block
        _norm("norm_8192x8192", 1, 8192, 8192, "bf16", "bf16", "none", True, False),
        # a training step: both norms, a learned gain for each channel of the branch
        _norm("norm_train_8192x4096", 4, 2048, 4096, "bf16", "f32", "channel", True, True),
        # odd sizes, a gate for each token and channel
        _norm("norm_train_5x411x1111", 5, 411, 1111, "f16", "f16", "token", False, True),
        # sixteen answers are scored by another model
        _head("head_16x32000x4096", 16, 32000, 4096, "bf16", False, False),
        # a training step that trains the head too
        _head("head_train_2048x32000x4096", 2048, 32000, 4096, "bf16", False, True, True),
        # the same under a large vocabulary: the largest products
        _head("head_train_4096x131072x4096", 4096, 131072, 4096, "bf16", False, True, False, 0.1),
        # odd sizes in fp16
        _head("head_train_777x50001x1000", 777, 50001, 1000, "f16", False, True, True, 0.2),
        # a training step above a packed head, which is frozen
        _head("head_packed_1024x32000x4096", 1024, 32000, 4096, "bf16", True, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "norm", "head", "head"])
    grad = rng.random() < 0.6
    if kind == "norm":
        width = rng.choice([64 * rng.randint(1, 8), 512 * rng.randint(1, 24), _log(rng, 64, 12000)])
        most = (MOST_NORM_GRAD if grad else MOST_NORM) // width
        rows = _log(rng, 1, min(16384, most))
        B = rng.choice([b for b in (1, 2, 3, 5, 8) if b <= rows])
        return {"kind": kind, "B": B, "T": rows // B, "width": width,
                "dt": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "wdt": rng.choice(["same", "f32"]),
                "gate": rng.choice(["none", "channel", "sequence", "token"]),
                "post": rng.random() < 0.5, "grad": grad}
    vocab = _log(rng, 1000, 131072)
    padded = rng.choice([0.0, 0.0, 0.1, 0.5])
    if kind == "embed":
        width = rng.choice([512 * rng.randint(1, 8), _log(rng, 64, 4096)])
        width = min(width, MOST_WEIGHTS // 2 // vocab)
        return {"kind": kind, "rows": _log(rng, 1, min(65536, MOST_EMBEDDED // width)),
                "vocab": vocab, "width": width, "dt": rng.choice(["bf16", "f16", "f32"]),
                "grad": grad, "padded": padded}
    packed = rng.random() < 0.25
    width = rng.choice([512 * rng.randint(1, 8), _log(rng, 64, 4096)])
    if packed:
        width = -(-width // 128) * 128
    rows = _log(rng, 1, min(8192, MOST_PRODUCT // (vocab * width)))
    return {"kind": kind, "rows": rows, "vocab": vocab, "width": width,
            "dt": rng.choice(["bf16", "f16"]), "packed": packed, "grad": grad,
            "entropy": rng.random() < 0.4, "padded": padded}


# ------------------------------------------------------------------ inputs
def _tokens(case, g):
    """Tokens as texts have them, a few of them often (the n-th most frequent one about 1/n of
    the time), their numbers in no order; a part of them is padding, -100."""
    n, V = case["rows"], case["vocab"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    t = (torch.exp(u * math.log(V)).long() - 1).clamp(0, V - 1)
    t = (t * 7919 + 13) % V if V % 7919 else t
    return torch.where(torch.rand(n, generator=g, device=DEV) < case["padded"], -100, t)


def _gains(g, width, dt):
    return (1 + 0.2 * torch.randn(width, generator=g, device=DEV)).to(dt)


def _prepare_embed(case, g):
    dt, n, V, K = DT[case["dt"]], case["rows"], case["vocab"], case["width"]
    s = {"tokens": _tokens(case, g), "scale": math.sqrt(K),
         "weight": (torch.randn(V, K, generator=g, device=DEV) / math.sqrt(K)).to(dt)}
    if case["grad"]:
        s["weight"].requires_grad_(True)
        s["g_out"] = (torch.randn(n, K, generator=g, device=DEV) / n).to(dt)
    return s


def _prepare_norm(case, g):
    dt, shape = DT[case["dt"]], (case["B"], case["T"], case["width"])
    wdt = DT.get(case["wdt"], dt)
    s = {"x": 2 * torch.randn(shape, generator=g, device=DEV),
         "branch": torch.randn(shape, generator=g, device=DEV)}
    s["x"][..., ::61] *= 8  # a few channels stand out
    s = {k: v.to(dt) for k, v in s.items()}
    s |= {"weight": _gains(g, case["width"], wdt), "scale": 0.7, "gate": None,
          "branch_weight": _gains(g, case["width"], wdt) if case["post"] else None}
    if case["gate"] == "channel":
        s["gate"] = (0.3 * torch.randn(case["width"], generator=g, device=DEV)).to(wdt)
    elif case["gate"] != "none":
        T = 1 if case["gate"] == "sequence" else case["T"]
        s["gate"] = torch.randn(case["B"], T, case["width"], generator=g, device=DEV).to(dt)
    if case["grad"]:
        for k in ("x", "branch", "weight", "gate", "branch_weight"):
            if s[k] is not None:
                s[k].requires_grad_(True)
        n = case["B"] * case["T"]
        s["g_stream"] = (torch.randn(shape, generator=g, device=DEV) / n).to(dt)
        s["g_normed"] = (torch.randn(shape, generator=g, device=DEV) / n).to(dt)
    return s


def _prepare_head(case, g):
    dt, n, V, K = DT[case["dt"]], case["rows"], case["vocab"], case["width"]
    s = {"tokens": _tokens(case, g)}
    # logits of a few units, the given token's higher than most
    if case["packed"]:
        s["codes"] = torch.randint(256, (V, K // 2), generator=g, device=DEV).to(torch.uint8)
        near = 127 + round(math.log2(1 / math.sqrt(K)))
        s["scales"] = torch.randint(near - 2, near + 1, (V, K // 32), generator=g,
                                    device=DEV).to(torch.uint8)
        w = _decoded(s["codes"], s["scales"])
        if own:  # packed once, on the host, as a program keeps it
            from if_i_could_turn_back_time_amd import PackedWeight
            s["packed"] = PackedWeight("e2m1", V, K, s["codes"].cpu(), s["scales"].cpu(),
                                       device=DEV)
    else:
        s["weight"] = w = (2.5 / math.sqrt(K) * torch.randn(V, K, generator=g, device=DEV)).to(dt)
    x = torch.randn(n, K, generator=g, device=DEV)
    at = w[s["tokens"].clamp(0, V - 1)].float()
    x += 4 * torch.rand(n, 1, generator=g, device=DEV) * at / at.norm(dim=-1, keepdim=True)
    s["hidden"] = x.to(dt)
    if case["grad"]:
        s["hidden"].requires_grad_(True)
        if not case["packed"]:
            s["weight"].requires_grad_(True)
        s["g_logprob"] = -(0.5 + torch.rand(n, generator=g, device=DEV)) / n
        s["g_entropy"] = None
        if case["entropy"]:
            s["g_entropy"] = -0.01 * torch.rand(n, generator=g, device=DEV) / n
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    make = {"embed": _prepare_embed, "norm": _prepare_norm, "head": _prepare_head}[case["kind"]]
    return {"kind": case["kind"], "grad": case["grad"], **make(case, g)}


# ------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)(state)


def _leaves(s, *names):
    return [k for k in names if s.get(k) is not None and s[k].requires_grad]


def _own(s):
    from if_i_could_turn_back_time_amd import head_logprobs, residual_norm, token_embedding
    if s["kind"] == "embed":
        out = token_embedding(s["tokens"], s["weight"], s["scale"])
        if not s["grad"]:
            return {"out": out}
        gw, = torch.autograd.grad(out, s["weight"], s["g_out"])
        return {"out": out.detach(), "grad_weight": gw}
    if s["kind"] == "norm":
        r = residual_norm(s["x"], s["weight"], s["branch"], gate=s["gate"], scale=s["scale"],
                          branch_weight=s["branch_weight"], eps=EPS)
        out = {"stream": r.stream.detach(), "normed": r.normed.detach()}
        if s["grad"]:
            names = _leaves(s, "x", "branch", "weight", "gate", "branch_weight")
            grads = torch.autograd.grad((r.stream, r.normed), [s[k] for k in names],
                                        (s["g_stream"], s["g_normed"]))
            out |= {"grad_" + k: v for k, v in zip(names, grads)}
        return out
    r = head_logprobs(s["hidden"], s.get("packed", s.get("weight")), s["tokens"])
    out = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach()}
    if s["grad"]:
        names = _leaves(s, "hidden", "weight")
        pairs = [(r.logprob, s["g_logprob"]), (r.entropy, s["g_entropy"])]
        of, with_ = zip(*[p for p in pairs if p[1] is not None])
        grads = torch.autograd.grad(of, [s[k] for k in names], with_)
        out |= {"grad_" + k: v for k, v in zip(names, grads)}
    return out


@torch.no_grad()
def _plain(s):
    return {"embed": _plain_embed, "norm": _plain_norm, "head": _plain_head}[s["kind"]](s)


def _plain_embed(s):
    w, V = s["weight"], s["weight"].shape[0]
    given = ((s["tokens"] >= 0) & (s["tokens"] < V))[:, None]
    at = s["tokens"].clamp(0, V - 1)
    out = {"out": torch.where(given, w[at].float() * s["scale"], 0.0).to(w.dtype)}
    if s["grad"]:
        gw = torch.zeros(w.shape, device=DEV)
        gw.index_add_(0, at, torch.where(given, s["g_out"].float(), 0.0))
        out["grad_weight"] = (gw * s["scale"]).to(w.dtype)
    return out


def _plain_norm(s):
    x, b, w = (s[k].float() for k in ("x", "branch", "weight"))
    g = 1.0 if s["gate"] is None else s["gate"].float()
    wb = None if s["branch_weight"] is None else s["branch_weight"].float()
    nb = b
    if wb is not None:
        r1 = torch.rsqrt(b.square().mean(-1, keepdim=True) + EPS)
        nb = b * r1
    b2 = nb if wb is None else nb * wb
    h = x + s["scale"] * g * b2
    r2 = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    n = h * r2
    dt = s["x"].dtype
    out = {"stream": h.to(dt), "normed": (n * w).to(dt)}
    if not s["grad"]:
        return out
    gy = s["g_normed"].float()
    dn = gy * w
    dx = s["g_stream"].float() + r2 * (dn - n * (dn * n).mean(-1, keepdim=True))
    t = s["scale"] * dx
    db = t * g
    grads = {"x": dx, "weight": (gy * n).sum((0, 1))}
    if s["gate"] is not None:
        dg = t * b2
        over = [i for i in range(3) if i >= 3 - s["gate"].dim() and s["gate"].shape[i - 3] == 1
                and dg.shape[i] > 1]
        over = [0, 1] if s["gate"].dim() == 1 else over
        grads["gate"] = dg.sum(over).reshape(s["gate"].shape) if over else dg
    if wb is not None:
        grads["branch_weight"] = (db * nb).sum((0, 1))
        db = db * wb
        db = r1 * (db - nb * (db * nb).mean(-1, keepdim=True))
    grads["branch"] = db
    for k in _leaves(s, "x", "branch", "weight", "gate", "branch_weight"):
        out["grad_" + k] = grads[k].to(s[k].dtype)
    return out


def _decoded(codes, scales):
    """[V, K] fp32 of packed E2M1 codes (element 2 j in the low half of byte j) and E8M0 scales."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    w = table[c].unflatten(-1, (-1, 32))
    return torch.ldexp(w, (scales.int() - 127)[..., None]).flatten(-2)


def _plain_head(s):
    x, tok = s["hidden"].float(), s["tokens"][:, None]
    w = s["weight"].float() if "weight" in s else _decoded(s["codes"], s["scales"])
    given = (tok >= 0) & (tok < w.shape[0])
    at = tok.clamp(0, w.shape[0] - 1)
    logp = x @ w.T
    logp -= logp.amax(-1, keepdim=True)
    logp -= logp.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    pl = p * logp
    entropy = -pl.sum(-1, keepdim=True)
    out = {"logprob": torch.where(given, logp.gather(1, at), 0.0)[:, 0], "entropy": entropy[:, 0]}
    if not s["grad"]:
        return out
    g = torch.where(given, s["g_logprob"][:, None], 0.0)
    d = p * -g
    if s["g_entropy"] is not None:
        d -= s["g_entropy"][:, None] * (pl + p * entropy)
    d.scatter_add_(1, at, g)
    out["grad_hidden"] = (d @ w).to(s["hidden"].dtype)
    if "weight" in s:
        out["grad_weight"] = (d.T @ x).to(s["weight"].dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 4 if case["dt"] == "f32" else 2
    K, grad = case["width"], case["grad"]
    if case["kind"] == "norm":
        n = case["B"] * case["T"] * K
        we = 4 if case["wdt"] == "f32" else e
        vectors = K * we * (1 + case["post"] + (case["gate"] == "channel"))
        per = {"sequence": case["B"] * K * e, "token": n * e}.get(case["gate"], 0)
        if not grad:
            return {"bytes": 4 * n * e + vectors + per, "flops": 10 * n}
        # x, the branch and two gradients read, two outputs and two gradients written
        return {"bytes": 8 * n * e + 2 * vectors + 2 * per, "flops": 40 * n}
    n, V = case["rows"], case["vocab"]
    if case["kind"] == "embed":
        if not grad:
            return {"bytes": n * (8 + 2 * K * e), "flops": n * K}
        return {"bytes": n * (8 + 3 * K * e) + V * K * e, "flops": 3 * n * K}
    w = V * K // 2 + V * K // 32 if case["packed"] else 2 * V * K
    if not grad:
        return {"bytes": w + n * (2 * K + 16), "flops": 2 * n * V * K}
    if case["packed"]:
        return {"bytes": w + n * (4 * K + 24), "flops": 4 * n * V * K}
    return {"bytes": 2 * w + n * (4 * K + 24), "flops": 6 * n * V * K}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_embed(case, s):
    w, tok, V = s["weight"].detach(), s["tokens"], case["vocab"]
    inside = torch.nonzero((tok >= 0) & (tok < V))[:, 0]
    out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device=DEV)
    out[inside] = w[tok[inside]].double() * s["scale"]
    if not case["grad"]:
        return {"out": out}
    gw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    gw.index_put_((tok[inside],), s["g_out"][inside].double(), accumulate=True)
    return {"out": out, "grad_weight": gw.mul_(s["scale"])}


def _exact_norm(case, s):
    """Outputs from the formulas, gradients by automatic differentiation of them."""
    names = [k for k in ("x", "branch", "weight", "gate", "branch_weight") if s[k] is not None]
    v = {k: s[k].detach().double().requires_grad_(case["grad"]) for k in names}
    with torch.enable_grad():
        b = v["branch"]
        if "branch_weight" in v:
            b = b / torch.sqrt((b * b).sum(-1, keepdim=True) / case["width"] + EPS)
            b = b * v["branch_weight"]
        if "gate" in v:
            b = b * v["gate"]
        h = v["x"] + s["scale"] * b
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["width"] + EPS) * v["weight"]
        out = {"stream": h.detach(), "normed": y.detach()}
        if case["grad"]:
            up = (s["g_stream"].double(), s["g_normed"].double())
            grads = torch.autograd.grad((h, y), [v[k] for k in names], up)
            out |= {"grad_" + k: g for k, g in zip(names, grads)}
    return out


def _exact_head(case, s):
    V, K, M = case["vocab"], case["width"], case["rows"]
    if case["packed"]:
        nibbles = torch.empty(V, K, dtype=torch.int64, device=DEV)
        nibbles[:, 0::2], nibbles[:, 1::2] = s["codes"] % 16, s["codes"] // 16
        m, sign = nibbles % 8, 1.0 - 2.0 * (nibbles // 8).double()
        e = (m // 2).clamp(min=1).double() - 1  # exponent 0 is the subnormal one
        w = sign * torch.where(m >= 2, 1 + 0.5 * (m % 2), 0.5 * (m % 2)) * torch.exp2(e)
        w *= torch.exp2(s["scales"].double() - 127).repeat_interleave(32, 1)
    else:
        w = s["weight"].detach().double()
    tok = s["tokens"]
    step = max(1, (1 << 28) // V)
    rows, gw = [], torch.zeros_like(w) if case["grad"] and not case["packed"] else None
    for r in range(0, M, step):
        x, t = s["hidden"].detach()[r:r + step].double(), tok[r:r + step]
        i = torch.nonzero((t >= 0) & (t < V))[:, 0]
        logp = torch.log_softmax(x @ w.T, -1)
        lp = torch.zeros(len(x), dtype=torch.float64, device=DEV)
        lp[i] = logp[i, t[i]]
        p = logp.exp()
        ent = -(p * logp).sum(-1)
        row = [lp, ent]
        if case["grad"]:
            up = torch.zeros_like(lp)
            up[i] = s["g_logprob"][r:r + step][i].double()
            coefficient = up[:, None]
            if s["g_entropy"] is not None:
                coefficient = coefficient + (s["g_entropy"][r:r + step, None].double()
                                             * (logp + ent[:, None]))
            d = p.mul_(coefficient).neg_()
            d[i, t[i]] += up[i]
            row.append(d @ w)
            if gw is not None:
                gw.addmm_(d.T, x)
        rows.append(row)
    out = dict(zip(("logprob", "entropy", "grad_hidden"), (torch.cat(c) for c in zip(*rows))))
    if gw is not None:
        out["grad_weight"] = gw
    return out


def exact(case, seed):
    s = prepare(case, seed)
    of = {"embed": _exact_embed, "norm": _exact_norm, "head": _exact_head}[case["kind"]]
    return of(case, s)
