"""CPU restatement in fp64 of the 8-bit key/value cache, attention over it, eviction from it and
the token log probabilities.  Test infrastructure only; shares no code with the package.

A cache here is a dict of one sequence's and head's blocks in a plain layout: codes as fp64 values
[tokens, D] and exponents [blocks]."""
from __future__ import annotations

import numpy as np

BLOCK = 32


def e4m3(x: np.ndarray) -> np.ndarray:
    """Rounded to the nearest E4M3 value, ties to even; not finite becomes NaN."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    a = np.where(ok, np.abs(x), 0.0)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.where(ok, np.copysign(np.rint(a / step) * step, x), np.nan)


def exponent(amax: float) -> int:
    """The least e >= -100 with amax <= 448 * 2^e."""
    e = -100
    while amax > np.ldexp(448.0, e):
        e += 1
    return e


def finite_max(x: np.ndarray) -> float:
    x = np.abs(x[np.isfinite(x)])
    return float(x.max()) if x.size else 0.0


class Tokens:
    """One head's keys (or values) of one sequence."""

    def __init__(self, D: int):
        self.codes = np.zeros((0, D))
        self.exps: list[int] = []

    def append(self, x: np.ndarray, start: int | None = None) -> None:
        x = np.asarray(x, np.float64)
        start = len(self.codes) if start is None else start
        self.codes = self.codes[:start]
        end = start + len(x)
        self.exps = self.exps[:(start + BLOCK - 1) // BLOCK]
        for b in range(start // BLOCK, (end + BLOCK - 1) // BLOCK):
            lo, hi = max(b * BLOCK, start), min((b + 1) * BLOCK, end)
            new = x[lo - start:hi - start]
            e = exponent(finite_max(new))
            if b * BLOCK < start:  # earlier tokens in the block
                e = max(e, self.exps[b])
                old = self.codes[b * BLOCK:start]
                if e > self.exps[b]:
                    self.codes[b * BLOCK:start] = e4m3(old * 2.0 ** (self.exps[b] - e))
                self.exps[b] = e
            else:
                self.exps.append(e)
            self.codes = np.concatenate([self.codes[:lo], e4m3(new * 2.0 ** -e)])

    def values(self) -> np.ndarray:
        e = np.repeat(np.asarray(self.exps, np.float64), BLOCK)[:len(self.codes)]
        return self.codes * 2.0 ** e[:, None]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """q [n, D] (a head's rows, the last n places), k, v [tokens, D] -> out [n, D], lse [n],
    p [n, tokens], and the sums that error bounds are made of: sum |q k|, sum p |v|."""
    n, t = len(q), len(k)
    out = np.zeros((n, v.shape[1]))
    lse = np.full(n, -np.inf)
    p = np.zeros((n, t))
    mags, pv = np.zeros(n), np.zeros((n, v.shape[1]))
    with np.errstate(invalid="ignore"):
        for i in range(n):
            sees = t - n + i + 1
            if sees <= 0:
                continue
            s = scale * (k[:sees] @ q[i])
            m = s.max()
            e = np.exp(s - m)
            z = e.sum()
            p[i, :sees] = e / z
            out[i] = p[i, :sees] @ v[:sees]
            lse[i] = m + np.log(z)
            mags[i] = scale * (np.abs(k[:sees]) @ np.abs(q[i])).max()
            pv[i] = p[i, :sees] @ np.abs(v[:sees])
    return out, lse, p, mags, pv


def evict(weights: np.ndarray, keep: int, recent: int) -> np.ndarray:
    """Places of one head's tokens (weights [tokens]) that stay, ascending."""
    n = len(weights)
    if n <= keep:
        return np.arange(n)
    m = n - recent
    w = np.where(np.isnan(weights[:m]), -np.inf, weights[:m].astype(np.float64))
    nan = np.isnan(weights[:m])
    order = sorted(range(m), key=lambda t: (nan[t], -w[t], t))
    return np.sort(np.concatenate([np.array(order[:keep - recent], np.int64),
                                   np.arange(m, n)]))


def logprobs(x: np.ndarray, token: int, top: int):
    """logprob, entropy, top logprobs and ids of one row, and p and log p."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max()
        if m == -np.inf:
            logp = np.full(len(x), -np.inf)
        else:
            logp = x - m - np.log(np.exp(x - m).sum())
        p = np.exp(logp)
        entropy = -np.where(p > 0, p * logp, 0.0).sum()
    nan = np.isnan(x)
    order = sorted(range(len(x)), key=lambda i: (not nan[i], 0.0 if nan[i] else -x[i], i))[:top]
    lp = logp[token] if 0 <= token < len(x) else 0.0
    return lp, entropy, logp[order], np.array(order, np.int64), p, logp


def logprobs_grad(p, logp, entropy, token, g_lp, g_ent, top_ids=(), g_top=()):
    """The formula's gradient of one row."""
    inside = 0 <= token < len(p)
    total = (g_lp if inside else 0.0) + float(np.sum(g_top))
    with np.errstate(invalid="ignore"):
        g = np.where(p > 0, -p * (total + g_ent * (logp + entropy)), 0.0)
    if inside:
        g[token] += g_lp
    for i, t in zip(top_ids, g_top):
        g[i] += t
    return g
