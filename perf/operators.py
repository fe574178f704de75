"""The operators a program needs around the 4-bit linear layer once it answers with a model:
writing keys and values into a cache held in 8 bits, attention over that cache, eviction from it
by accumulated attention weight, and the log probabilities of given tokens (with the gradient).

``listed`` holds the cases that are timed and ``draw`` gives more of the same ranges.  With
``own`` false a pass computes the operator in plain fp32 torch operations, with it true it makes
the framework's calls; both work on the tensors that ``prepare`` makes.

The cache: pages of P tokens (P a multiple of 32), all heads of a page together.

    k        float8_e4m3fn [pages, heads, P, D]
    v        float8_e4m3fn [pages, heads, P / 16, D, 16]    16 tokens of one channel side by side
    k_scale  uint8 [pages, heads, P / 32]                   2^(s - 127), one for each block of
    v_scale  (the same)                                     32 tokens and head
    table    int32 [sequences, most pages]                  a sequence's pages in order

A block's scale is the least power of two, from 2^-100 up, that brings its largest value to at
most 448, the largest of E4M3.  A block that is appended to keeps the larger of its scale and
the new tokens' own; where it grows, the earlier tokens' codes are rounded to the new one.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK, SIDE = 32, 16
F8 = torch.float8_e4m3fn
MOST_SCORES = 64 * 4096 * 4096   # query rows x cached tokens of the largest listed prompt
MOST_CACHED = 2 * 8 * 100003     # tokens x heads of the largest listed cache that is read
MOST_LOGITS = 1024 * 131072


def _attend(name, B, hq, hkv, D, page, new, length, dt, weights=False):
    return {"name": name, "kind": "attend", "B": B, "hq": hq, "hkv": hkv, "D": D, "page": page,
            "new": new, "len": length, "dt": dt, "weights": weights}


def listed():
    return [
        # one decoded token of one sequence enters the cache (4096 wide: 32 heads of 128); all
        # launch cost
        {"name": "append_b1_1", "kind": "append", "B": 1, "hkv": 32, "D": 128, "page": 64,
         "new": 1, "len": 777, "dt": "f16"},
        # four prompts of up to 2048 tokens enter it (8192 wide, 8 shared heads), two of them
        # behind an earlier part that ends inside a block
        {"name": "append_b4_2048", "kind": "append", "B": 4, "hkv": 8, "D": 128, "page": 64,
         "new": 2048, "len": 3000, "dt": "bf16"},
        # one token decoded over a short cache, a head of its own for each query head
        _attend("attend_b1_777", 1, 32, 32, 128, 64, 1, 777, "f16"),
        # sixteen sequences of different lengths decoded together, 8 query heads to a cached
        # one; the weights are summed up for the eviction
        _attend("attend_b16_8192_w", 16, 64, 8, 128, 64, 1, 8192, "bf16", True),
        # two sequences over a long context: the largest read of a cache
        _attend("attend_b2_100003", 2, 64, 8, 128, 128, 1, 100003, "bf16"),
        # the next part of two prompts, odd lengths, behind what the cache holds of them
        _attend("attend_part_333_of_4001", 2, 32, 32, 128, 64, 333, 4001, "f16"),
        # a whole prompt of 4096 tokens: the largest product
        _attend("attend_prompt_4096", 1, 64, 8, 128, 64, 4096, 4096, "bf16"),
        # one sequence's cache is cut to a quarter
        {"name": "evict_b1_4096_1024", "kind": "evict", "B": 1, "hkv": 32, "D": 128, "page": 64,
         "len": 4096, "keep": 1024, "recent": 128},
        # sixteen sequences of different lengths at once
        {"name": "evict_b16_8192_2048", "kind": "evict", "B": 16, "hkv": 8, "D": 128, "page": 64,
         "len": 8192, "keep": 2048, "recent": 256},
        # sixteen sampled tokens with their five likeliest alternatives, part of the vocabulary
        # forbidden
        {"name": "logprobs_16x32000_top5", "kind": "logprobs", "rows": 16, "vocab": 32000,
         "top": 5, "dt": "f16", "forbid": True, "grad": False},
        # a text's tokens scored under a large vocabulary, with twenty alternatives each
        {"name": "logprobs_1024x131072_top20", "kind": "logprobs", "rows": 1024,
         "vocab": 131072, "top": 20, "dt": "bf16", "forbid": False, "grad": False},
        # a training step's loss: log probabilities and entropies of a batch, and the gradient
        {"name": "train_2048x32000", "kind": "logprobs", "rows": 2048, "vocab": 32000, "top": 0,
         "dt": "bf16", "forbid": False, "grad": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "evict",
                       "logprobs", "logprobs"])
    dt = rng.choice(["f16", "bf16"])
    if kind == "logprobs":
        grad = rng.random() < 0.4
        vocab = _log(rng, 1000, 131072)
        rows = _log(rng, 1, min(4096, MOST_LOGITS // vocab // (4 if grad else 1)))
        return {"kind": kind, "rows": rows, "vocab": vocab,
                "top": 0 if grad else rng.choice([0, 1, 5, 8, 20]),
                "dt": rng.choice(["f16", "bf16", "bf16", "f32"]), "forbid": rng.random() < 0.3,
                "grad": grad}
    B = rng.choice([1, 1, 2, 3, 5, 8, 16, 24])
    hkv, group = rng.choice([1, 2, 4, 8, 8, 12, 32]), rng.choice([1, 1, 2, 4, 5, 8])
    if hkv * group > 64:
        group = 2
    D, page = rng.choice([64, 128, 128, 128, 256]), rng.choice([32, 64, 64, 128, 256])
    most = max(600, min(100000, MOST_CACHED * 128 // (B * hkv * D)))
    case = {"kind": kind, "B": B, "hkv": hkv, "D": D, "page": page}
    if kind == "evict":
        length = _log(rng, 300, min(32768, max(301, most // 2)))
        keep = _log(rng, 40, length)
        return case | {"len": length, "keep": keep, "recent": rng.randint(0, keep // 2)}
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, max(3, min(4096, most // 4)))])
        return case | {"new": new, "len": new + _log(rng, 1, 4000), "dt": dt}
    new = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 4096), _log(rng, 9, 4096)])
    length = _log(rng, 64, min(most, max(65, MOST_SCORES // (B * hkv * group * new))))
    return case | {"hq": hkv * group, "new": min(new, length), "len": length, "dt": dt,
                   "weights": rng.random() < 0.25}


# ------------------------------------------------------------------ inputs
def _spread(case, key):
    """Whole numbers for the sequences of a case: the first has case[key], the others from half
    of that on."""
    rng = random.Random("%s %s" % (key, sorted((k, v) for k, v in case.items() if k != "name")))
    most = case[key]
    return [most] + [rng.randint(max(1, most // 2), most) for _ in range(case["B"] - 1)]


def _lens(case):
    """What a sequence holds after the call, and how many of these tokens are the call's own."""
    held = _spread(case, "len")
    if "new" not in case:
        return held, None
    new = [min(n, t) for n, t in zip(_spread(case, "new"), held)]
    if case["kind"] == "append":  # every other prompt is its sequence's first part
        held = [n if n > 1 and i % 2 == 0 else t for i, (n, t) in enumerate(zip(new, held))]
    return held, new


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _byte(amax):
    """The scale byte of a block whose largest magnitude is amax (fp32)."""
    m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e.clamp(min=-100), -100) + 127


def _filled(g, pages, heads, page, D):
    """A pool of pages as appending normally distributed keys and values leaves it."""
    x = torch.randn(pages, heads, page // BLOCK, BLOCK, D, generator=g, device=DEV)
    x[..., ::37] *= 3  # a few channels stand out
    s = _byte(x.abs().amax((-1, -2)))
    codes = torch.ldexp(x, (127 - s)[..., None, None]).to(F8)
    return codes, s.to(torch.uint8)


def _cache(case, g, extra=0):
    """The four tensors of a cache, and the page table of its sequences: pages in no order."""
    B, page = case["B"], case["page"]
    per = -(-case["len"] // page)
    pages = B * (per + extra)
    k, ks = _filled(g, pages, case["hkv"], page, case["D"])
    v, vs = _filled(g, pages, case["hkv"], page, case["D"])
    table = torch.randperm(pages, generator=g, device=DEV).int().reshape(B, per + extra)
    k = k.reshape(pages, case["hkv"], page, case["D"])
    v = v.view(torch.uint8).view(pages, case["hkv"], page // SIDE, SIDE, -1)
    v = v.transpose(-1, -2).contiguous().view(F8)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    if kind == "logprobs":
        M, V = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(M, V, generator=g, device=DEV)
        tokens = torch.randint(V, (M,), generator=g, device=DEV)
        x.scatter_add_(1, tokens[:, None], 4 * torch.rand(M, 1, generator=g, device=DEV))
        if case["forbid"]:
            x[:, torch.rand(V, generator=g, device=DEV) < 0.2] = float("-inf")
        state = {"kind": kind, "logits": x.to(DT[case["dt"]]), "tokens": tokens,
                 "top": case["top"]}
        if case["grad"]:
            state["logits"].requires_grad_(True)
            state["g_logprob"] = -(0.5 + torch.rand(M, generator=g, device=DEV)) / M
            state["g_entropy"] = -0.01 * torch.rand(M, generator=g, device=DEV) / M
        return state
    held, new = _lens(case)
    if kind == "evict":
        kept = -(-case["keep"] // case["page"])
        state = {"kind": kind, **_cache(case, g, kept), "lens": _int(held), "keep": case["keep"],
                 "recent": case["recent"], "max_len": case["len"], "held": held}
        state["new_table"] = state["table"][:, -kept:].contiguous()
        state["table"] = state["table"][:, :-kept].contiguous()
        # heavy tailed, and rounded so that some are equal
        w = torch.rand(case["B"], case["hkv"], case["len"], generator=g, device=DEV)
        state["weights"] = torch.round(64 * (1 / (w + 0.01))) / 64
        return state
    T, dt = sum(new), DT[case["dt"]]
    cu = _int([0] + torch.tensor(new).cumsum(0).tolist())
    state = {"kind": kind, **_cache(case, g), "cu": cu, "max_new": case["new"],
             "max_len": case["len"], "new": new, "held": held}
    if kind == "append":
        x = torch.randn(T, 2, case["hkv"], case["D"], generator=g, device=DEV)
        x[..., ::37] *= 3
        x = x.to(dt)
        # slices of one projection's output
        return state | {"xk": x[:, 0], "xv": x[:, 1],
                        "start": _int([t - n for t, n in zip(held, new)])}
    q = torch.randn(T, case["hq"], case["D"], generator=g, device=DEV).to(dt)
    state |= {"q": q, "lens": _int(held), "weights": None}
    if case["weights"]:
        state["weights"] = torch.rand(case["B"], case["hkv"], case["len"], generator=g,
                                      device=DEV)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from if_i_could_turn_back_time_amd import (KVCache, cache_append, cache_attention,
                                               cache_evict, token_logprobs)
    kind = s["kind"]
    if kind == "logprobs":
        r = token_logprobs(s["logits"], s["tokens"], top=s["top"])
        if "g_logprob" not in s:
            return {"logprob": r.logprob, "entropy": r.entropy, "top_logprobs": r.top_logprobs,
                    "top_ids": r.top_ids}
        gx, = torch.autograd.grad((r.logprob, r.entropy), (s["logits"],),
                                  (s["g_logprob"], s["g_entropy"]))
        return {"logprob": r.logprob.detach(), "entropy": r.entropy.detach(), "grad": gx}
    cache = KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "append":
        cache_append(cache, s["xk"], s["xv"], s["table"], s["start"], s["cu"],
                     max_new=s["max_new"])
        return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}
    if kind == "evict":
        r = cache_evict(cache, s["table"], s["lens"], s["weights"], s["keep"], s["recent"],
                        s["new_table"], max_len=s["max_len"])
        return {"kept": r.kept, "lens": r.lens, "weights": r.weights,
                **{n: s[n] for n in ("k", "v", "k_scale", "v_scale")}}
    out, lse = cache_attention(s["q"], cache, s["table"], s["lens"], s["cu"],
                               max_new=s["max_new"], max_len=s["max_len"], weights=s["weights"],
                               return_lse=True)
    return {"out": out, "lse": lse, "weights": s["weights"]}


def _plain(s):
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict,
            "logprobs": _plain_logprobs}[s["kind"]](s)


def _tokens(s, name, table):
    """[B, heads, tokens, D] of fp32 codes and [B, heads, tokens / 32] of exponents: what the
    pages of a table hold."""
    x = s[name][table.long()]
    if name == "v":
        x = x.float().transpose(-1, -2)
    B, n, h = x.shape[:3]
    x = x.float().reshape(B, n, h, -1, s["k"].shape[-1]).transpose(1, 2)
    e = s[name + "_scale"][table.long()].int().transpose(1, 2) - 127
    return x.reshape(B, h, -1, x.shape[-1]), e.reshape(B, h, -1)


def _put(s, name, codes, byte, at, page_of):
    """Writes blocks [n, heads, 32, D] of fp32 codes and their bytes at (page, block) pairs."""
    b = codes.to(F8).view(torch.uint8)
    if name == "v":
        pages, h, n, D, _ = s["v"].shape
        s["v"].view(torch.uint8).view(pages, h, n // 2, 2, D, SIDE)[page_of, :, at] = \
            b.view(*b.shape[:2], 2, SIDE, D).transpose(-1, -2)
    else:
        pages, h, page, D = s["k"].shape
        s["k"].view(torch.uint8).view(pages, h, page // BLOCK, BLOCK, D)[page_of, :, at] = b
    s[name + "_scale"][page_of, :, at] = byte.to(torch.uint8)


def _plain_append(s):
    start, cu, table = s["start"].long(), s["cu"].long(), s["table"].long()
    per = s["k"].shape[2] // BLOCK
    end = start + cu[1:] - cu[:-1]
    # the blocks that get tokens
    blk = (start // BLOCK)[:, None] + torch.arange((s["max_new"] + 30) // BLOCK + 1, device=DEV)
    seq, col = torch.nonzero((blk * BLOCK < end[:, None]) & (start < end)[:, None], as_tuple=True)
    blk = blk[seq, col]
    page_of, at = table[seq, blk // per], blk % per
    pos = blk[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    fresh = (pos >= start[seq, None]) & (pos < end[seq, None])
    row = torch.where(fresh, cu[seq, None] + pos - start[seq, None], 0)
    fresh = fresh[:, None, :, None]
    kept = (blk * BLOCK < start[seq])[:, None]
    for name, x in (("k", s["xk"]), ("v", s["xv"])):
        if name == "v":
            was = s["v"].view(*s["v"].shape[:2], per, 2, -1, SIDE)[page_of, :, at].float()
            was = was.transpose(-1, -2).flatten(2, 3)
        else:
            was = s["k"].view(*s["k"].shape[:2], per, BLOCK, -1)[page_of, :, at].float()
        byte = s[name + "_scale"][page_of, :, at].int()
        x = x[row].float().transpose(1, 2)
        need = _byte(torch.where(fresh, x.abs(), 0.0).amax((-1, -2)))
        to = torch.where(kept, torch.maximum(byte, need), need)
        old = torch.where(kept[..., None, None], torch.ldexp(was, (byte - to)[..., None, None]),
                          was)
        old = torch.where((pos < end[seq, None])[:, None, :, None], old, was)
        _put(s, name, torch.where(fresh, torch.ldexp(x, (127 - to)[..., None, None]), old), to,
             at, page_of)
    return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}


def _plain_attend(s):
    B, (hkv, D) = len(s["new"]), (s["k"].shape[1], s["k"].shape[3])
    T, most, cu = s["q"].shape[0], s["max_new"], s["cu"].long()
    group = s["q"].shape[1] // hkv
    (k, ek), (v, ev) = _tokens(s, "k", s["table"]), _tokens(s, "v", s["table"])
    n, t = k.shape[2], torch.arange(k.shape[2], device=DEV)
    held = t < s["lens"][:, None]
    k = torch.ldexp(k, ek.repeat_interleave(BLOCK, -1)[..., None])
    v = torch.ldexp(v, ev.repeat_interleave(BLOCK, -1)[..., None])
    k, v = (torch.where(held[:, None, :, None], x, 0.0) for x in (k, v))
    i = torch.arange(most, device=DEV)
    count = (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[rows].view(B, most, hkv, group, D).permute(0, 2, 3, 1, 4)
    sees = t <= (s["lens"][:, None] - count + i)[..., None]
    sees = (sees & held[:, None] & (i < count)[..., None])[:, None].repeat(1, group, 1, 1)
    sees = sees.view(B, 1, group * most, n)
    p = q.reshape(B, hkv, group * most, D) @ k.transpose(-1, -2)
    p = (p / math.sqrt(D)).masked_fill_(~sees, float("-inf"))
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    lse = m + l.log()
    p = p.div_(torch.where(l == 0, 1.0, l))
    out = (p @ v).view(B, hkv, group, most, D).permute(0, 3, 1, 2, 4).reshape(B, most, -1, D)
    lse = lse.view(B, hkv, group, most).permute(0, 3, 1, 2).reshape(B, most, -1)
    valid = (i < count)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)[..., :s["weights"].shape[-1]]
    return {"out": out[valid].to(s["q"].dtype), "lse": lse[valid], "weights": s["weights"]}


def _plain_evict(s):
    w, lens, keep = s["weights"], s["lens"].long()[:, None, None], s["keep"]
    n = w.shape[-1]
    t = torch.arange(n, device=DEV)
    score = torch.where(t >= lens - s["recent"], float("inf"), w)
    score = torch.where(t < lens, score, float("-inf"))
    if keep > n:
        score = torch.nn.functional.pad(score, (0, keep - n), value=float("-inf"))
    ids = score.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    ids = torch.where(ids < lens, ids, 1 << 30).sort(-1).values
    held = ids < 1 << 30
    kept = torch.where(held, ids, -1).int()
    safe = torch.where(held, ids, 0)
    weights = torch.where(held, w.gather(-1, safe.clamp(max=n - 1)), 0.0)
    B, h, per = *w.shape[:2], s["k"].shape[2] // BLOCK
    pad = -keep % BLOCK
    blocks = (keep + pad) // BLOCK
    seq, blk = (x.reshape(-1) for x in torch.meshgrid(
        torch.arange(B, device=DEV), torch.arange(blocks, device=DEV), indexing="ij"))
    full = (blk * BLOCK < s["lens"][seq].clamp(max=keep))
    seq, blk = seq[full], blk[full]
    page_of, at = s["new_table"].long()[seq, blk // per], blk % per
    there = torch.nn.functional.pad(held, (0, pad)).view(B, h, blocks, BLOCK, 1)
    for name in ("k", "v"):
        x, e = _tokens(s, name, s["table"])
        e = e.gather(-1, safe // BLOCK)
        x = x.gather(2, safe[..., None].expand(-1, -1, -1, x.shape[-1]))
        x = torch.nn.functional.pad(torch.where(held[..., None], torch.ldexp(x, e[..., None]),
                                                0.0), (0, 0, 0, pad))
        x = x.view(B, h, blocks, BLOCK, -1)
        to = _byte(x.abs().amax((-1, -2)))
        x = torch.where(there, torch.ldexp(x, (127 - to)[..., None, None]), 0.0)
        _put(s, name, x[seq, :, blk], to[seq, :, blk], at, page_of)
    return {"kept": kept, "lens": s["lens"].clamp(max=keep), "weights": weights,
            **{n: s[n] for n in ("k", "v", "k_scale", "v_scale")}}


def _plain_logprobs(s):
    x, tok = s["logits"].detach().float(), s["tokens"][:, None]
    m = x.amax(-1, keepdim=True)
    d = x - m
    p = d.exp()
    z = p.sum(-1, keepdim=True)
    p = p / z
    logp = d - z.log()
    pl = torch.where(p > 0, p * logp, 0.0)
    entropy = -pl.sum(-1, keepdim=True)
    logprob = logp.gather(1, tok)
    if "g_logprob" in s:
        g1, g2 = s["g_logprob"][:, None], s["g_entropy"][:, None]
        grad = -g1 * p - g2 * (pl + p * entropy)
        grad.scatter_add_(1, tok, g1)
        return {"logprob": logprob[:, 0], "entropy": entropy[:, 0],
                "grad": grad.to(s["logits"].dtype)}
    top = x.sort(dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    return {"logprob": logprob[:, 0], "entropy": entropy[:, 0],
            "top_logprobs": logp.gather(1, top), "top_ids": top}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n, e = case["rows"] * case["vocab"], 4 if case["dt"] == "f32" else 2
        out = case["rows"] * (8 + 8 + 12 * case["top"])
        # the row's values once, and with a gradient once more to write it
        return {"bytes": n * e * (2 if case["grad"] else 1) + out,
                "flops": n * (12 if case["grad"] else 5)}
    held, new = _lens(case)
    h, D = case["hkv"], case["D"]
    if kind == "evict":
        cut = sum(min(t, case["keep"]) for t in held) * h
        # every weight, then the kept keys and values from page to page with ids and weights
        return {"bytes": 4 * h * sum(held) + cut * (4 * D + 8), "flops": 6 * cut * D}
    if kind == "append":
        rows = sum(new) * h
        return {"bytes": rows * D * 2 * (2 + 1) + rows * 2 // BLOCK, "flops": 6 * rows * D}
    seen = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, held))
    b = sum(held) * h * (2 * D + 2 / BLOCK + (8 if case["weights"] else 0))
    b += sum(new) * case["hq"] * (4 * D + 4)
    return {"bytes": int(b), "flops": 4 * seen * case["hq"] * D}


# ------------------------------------------------------------------ the same in 64 bits
def _pages64(s, name, b):
    """Sequence b's keys or values, [heads, tokens, D] in fp64."""
    at = s["table"][b].long()
    x = s[name][at].double()
    if name == "v":
        x = x.transpose(-1, -2).flatten(2, 3)
    scale = torch.exp2(s[name + "_scale"][at].double() - 127).repeat_interleave(BLOCK, 2)
    return (x * scale[..., None]).transpose(0, 1).flatten(1, 2)


def _e4m3(x):
    """x rounded to the nearest E4M3 value, ties to even: 4 significant bits down to 2^-6, steps
    of 2^-9 below."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _quantised64(x, least=None):
    """Codes [heads, tokens, D] and exponents [heads, blocks] of a sequence's tokens from a block's
    start on; `least`: what the first block's exponent is at least."""
    h, n, D = x.shape
    x = torch.nn.functional.pad(x, (0, 0, 0, -n % BLOCK)).view(h, -1, BLOCK, D)
    amax = x.abs().amax((-1, -2))
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -100) / 448)).clamp(min=-100)
    if least is not None:
        e[:, 0] = torch.maximum(e[:, 0], least)
    return _e4m3(x / torch.exp2(e)[..., None, None]).view(h, -1, D)[:, :n], e


def _written64(s, pool, name, pages, first, codes, e):
    """Puts a sequence's codes, from token `first` on, into the copy of the pool."""
    per, pos = s["k"].shape[2], torch.arange(first, first + codes.shape[1], device=DEV)
    page, at, codes = pages[pos // per].long(), pos % per, codes.transpose(0, 1)
    if name == "k":
        pool["k"][page, :, at] = codes
    else:
        pool["v"][page, :, at // SIDE, :, at % SIDE] = codes
    pool[name + "_scale"][page, :, at // BLOCK] = e.transpose(0, 1).repeat_interleave(
        BLOCK, 0)[:len(pos)].to(torch.uint8) + 127


def _exact_pool(s):
    """The cache after an append or an eviction, from the definition."""
    names = ("k", "v", "k_scale", "v_scale")
    pool = {n: s[n].double() if n in ("k", "v") else s[n].clone() for n in names}
    more = {"kept": [], "weights": []}
    for b in range(len(s["held"])):
        n = s["held"][b]
        if s["kind"] == "evict":
            recent, keep = s["recent"], min(n, s["keep"])
            w = s["weights"][b, :, :n].double()
            early = w[:, :max(0, n - recent)].sort(dim=-1, descending=True, stable=True).indices
            ids = torch.cat([early[:, :max(0, keep - recent)], torch.arange(
                max(0, n - recent), n, device=DEV).expand(len(w), -1)], 1).sort(-1).values
            pad = (0, s["keep"] - keep)
            more["kept"].append(torch.nn.functional.pad(ids, pad, value=-1).int())
            more["weights"].append(torch.nn.functional.pad(w.gather(1, ids), pad))
        for name in ("k", "v"):
            x = _pages64(s, name, b)[:, :n]
            if s["kind"] == "evict":
                x = x.gather(1, ids[..., None].expand(-1, -1, x.shape[-1]))
                # the last block is written whole
                codes, e = _quantised64(torch.nn.functional.pad(x, (0, 0, 0, -keep % BLOCK)))
                _written64(s, pool, name, s["new_table"][b], 0, codes, e)
                continue
            at, start = int(s["cu"][b]), n - s["new"][b]
            first = start // BLOCK * BLOCK
            fresh = s["x" + name][at:at + s["new"][b]].double().transpose(0, 1)
            if first < start:
                per = s["k"].shape[2]
                old = s[name + "_scale"][s["table"][b, first // per].long(), :,
                                         first % per // BLOCK].double() - 127
                # the earlier tokens never ask for more than their block's own scale
                x = torch.cat([x[:, first:start], fresh], 1)
            else:
                x, old = fresh, None
            codes, e = _quantised64(x, old)
            _written64(s, pool, name, s["table"][b], first, codes, e)
    if s["kind"] == "evict":
        return {"kept": torch.stack(more["kept"]), "weights": torch.stack(more["weights"]),
                "lens": s["lens"].clamp(max=s["keep"]), **pool}
    return pool


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        rows = []
        x, tok = s["logits"].detach(), s["tokens"]
        step = max(1, (1 << 27) // case["vocab"])
        for r in range(0, case["rows"], step):
            logp = torch.log_softmax(x[r:r + step].double(), -1)
            p = logp.exp()
            ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
            lp = logp.gather(1, tok[r:r + step, None])[:, 0]
            if case["grad"]:
                g1, g2 = (s[n][r:r + step, None].double() for n in ("g_logprob", "g_entropy"))
                gx = -p * (g1 + g2 * (torch.where(p > 0, logp, 0.0) + ent[:, None]))
                last = gx.scatter_add_(1, tok[r:r + step, None], g1)
            else:  # equal values are equal here too, whichever of them is meant
                last = logp.topk(case["top"], -1).values
            rows.append((lp, ent, last))
        lp, ent, last = (torch.cat(v) for v in zip(*rows))
        if case["grad"]:
            return {"logprob": lp, "entropy": ent, "grad": last}
        return {"logprob": lp, "entropy": ent, "top_logprobs": last, "top_ids": None}
    if kind in ("append", "evict"):  # codes are what the definition rounds them to
        return _exact_pool(s)
    held, new = s["held"], s["new"]
    hkv, D = case["hkv"], case["D"]
    group = case["hq"] // hkv
    if case["B"] * case["hq"] * case["new"] * case["len"] > 2 * MOST_SCORES:
        return None
    out = torch.empty(sum(new), case["hq"], D, dtype=torch.float64, device=DEV)
    lse = torch.empty(sum(new), case["hq"], dtype=torch.float64, device=DEV)
    weights = None if s["weights"] is None else s["weights"].double()
    row = 0
    for b in range(case["B"]):
        n, t = new[b], held[b]
        k, v = (_pages64(s, x, b)[:, :t] for x in ("k", "v"))
        hidden = torch.arange(t, device=DEV) > torch.arange(t - n, t, device=DEV)[:, None]
        for h in range(hkv):
            for j in range(h * group, (h + 1) * group):
                a = s["q"][row:row + n, j].double() @ k[h].T / math.sqrt(D)
                a = a.masked_fill(hidden, float("-inf"))
                lse[row:row + n, j] = a.logsumexp(-1)
                a = torch.softmax(a, -1)
                out[row:row + n, j] = a @ v[h]
                if weights is not None:
                    weights[b, h, :t] += a.sum(0)
        row += n
    return {"out": out, "lse": lse, "weights": weights}
