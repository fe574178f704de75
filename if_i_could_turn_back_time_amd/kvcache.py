"""A key/value cache held in 8 bits, attention over it and eviction from it: what a model of
packed linear layers (``QuantLinear``) needs between them to answer.  The reference has no
attention; these operators have no counterpart there.

Keys and values are E4M3 codes with one power-of-two scale per 32 tokens and head, half the
bytes of a 16-bit cache.  They lie in pages that all sequences share: a sequence's tokens are in
the pages its row of an int32 ``table`` names, in order, and its length is an entry of an int32
tensor on the GPU.  Who owns which page is the program's business.  Nothing on the GPU is read
back, so every call can be captured in a HIP graph (``torch.cuda.graph``) and replayed while the
tables and lengths change.  The calls are no torch operators: tracing and recording them
(``torch.jit.trace``, ``make_fx``) is refused.

    cache = KVCache.new(pages=512, heads=8, head_dim=128)
    cache_append(cache, k, v, table, held)                  # one new token a sequence
    y = cache_attention(q, cache, table, held + 1)
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi as C

BLOCK = 32  # tokens of one scale
SIDE = 16   # tokens of one channel side by side in v


class KVCache(NamedTuple):
    """The pool of pages (``include/fourbit.h``): four contiguous tensors on one GPU.

    ``k`` float8_e4m3fn [pages, heads, page, D]; ``v`` float8_e4m3fn
    [pages, heads, page / 16, D, 16]; ``k_scale`` and ``v_scale`` uint8 [pages, heads, page / 32],
    2^(s - 127) for a block of 32 tokens.  D is a multiple of 16 up to 256, a page a multiple
    of 32 tokens."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def new(cls, pages: int, heads: int, head_dim: int, page: int = 64,
            device="cuda") -> "KVCache":
        """An empty pool."""
        if page < BLOCK or page % BLOCK:
            raise ValueError(f"a page is a multiple of {BLOCK} tokens, got {page}")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {head_dim}")
        f8 = {"dtype": torch.float8_e4m3fn, "device": device}
        u8 = {"dtype": torch.uint8, "device": device}
        return cls(torch.zeros(pages, heads, page, head_dim, **f8),
                   torch.zeros(pages, heads, page // SIDE, head_dim, SIDE, **f8),
                   torch.zeros(pages, heads, page // BLOCK, **u8),
                   torch.zeros(pages, heads, page // BLOCK, **u8))

    @property
    def page(self) -> int:
        """Tokens of a page."""
        return self.k.shape[2]

    def read(self, table: torch.Tensor, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values [heads, length, D] in fp32 that the pages of one sequence
        (``table``: its row) hold; for inspection, not a fast path."""
        at = table.long()
        n, H, P, D = self.k[at].shape
        k = self.k[at].float().view(n, H, P, D)
        v = self.v[at].float().transpose(-1, -2).reshape(n, H, P, D)
        out = []
        for x, s in ((k, self.k_scale), (v, self.v_scale)):
            s = s[at].int().repeat_interleave(BLOCK, 2)[..., None]
            # 2^(s - 127) from its bits: torch.ldexp takes a power, which the GPU rounds
            scale = torch.where(s > 0, s << 23, 1 << 22).int().view(torch.float32)
            out.append((x * scale).transpose(0, 1).reshape(H, n * P, D)[:, :length])
        return out[0], out[1]


class Evicted(NamedTuple):
    """What :func:`cache_evict` returns."""
    kept: torch.Tensor     # int32 [sequences, heads, keep]: places kept, ascending, then -1
    lens: torch.Tensor     # int32 [sequences]: min(length, keep)
    weights: torch.Tensor  # fp32 [sequences, heads, keep]: their weights, then 0


def cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                 start: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                 max_new: int | None = None) -> None:
    """Writes new keys and values [tokens, heads, D] (fp16, bf16 or fp32; any strides between
    tokens and heads) into the cache, sequence b's from place ``start[b]`` on.

    ``cu_seqlens`` (int32 [sequences + 1]): sequence b's tokens are rows ``cu_seqlens[b]`` to
    ``cu_seqlens[b + 1]``; without it there is one token a sequence.  ``max_new``: the most new
    tokens of one sequence (those behind its first ``max_new`` are not written); by default all
    of them could be one's.

    A block's scale is the least power of two (from 2^-100 up) that brings its values within
    E4M3's range; values are rounded to nearest even, non-finite ones are held as NaN.  A block
    that holds earlier tokens keeps the larger scale, and where that grows the earlier codes are
    rounded to it.  Tokens beyond a sequence's pages are not written."""
    C.native().cache_append(*cache, k, v, table, start, cu_seqlens, max_new)


def cache_attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lens: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, *, max_new: int | None = None,
                    max_len: int | None = None, scale: float | None = None,
                    weights: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale * q k^T) v over the cache: [tokens, query heads, D] of q's dtype (fp16 or
    bf16), with fp32 sums.  The query heads are a multiple of the cache's; consecutive ones share
    a cached head.  ``scale`` is 1 / sqrt(D) by default.

    ``lens`` (int32 [sequences]) counts the tokens held, the new ones among them: row i of a
    sequence's n new rows sees the first ``lens - n + i + 1`` tokens.  A row that sees none gets
    0 (and an lse of -inf), and so does one that is no sequence's (in front of ``cu_seqlens[0]`` or
    from its last entry on, as in a batch padded for a graph).  A value of a token that a row does not see never reaches it, NaN or
    not.  ``cu_seqlens`` and ``max_new`` as for :func:`cache_append` (``max_new`` too small
    changes speed only, except that ``weights`` may miss the rows beyond it); ``max_len``: about
    the longest length, by which the work is split.  One sequence, and more than 64, should have it
    close: 8,000 tokens of 32 heads take 18 us under their own length and 118 under 131,072 (2 to 64
    sequences are dealt out by their lengths).

    ``weights`` (fp32 [sequences, heads, at least max_len]): grows in place by the attention
    weight that each held token got in this call, summed over rows and query heads; what
    :func:`cache_evict` goes by.  ``return_lse``: also the log of the sum of exponentials, fp32
    [tokens, query heads].  There is no gradient."""
    out, lse = C.native().cache_attention(q, *cache, table, lens, cu_seqlens, max_new, max_len,
                                          scale, weights, return_lse)
    return (out, lse) if return_lse else out


def cache_evict(cache: KVCache, table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor,
                keep: int, recent: int, new_table: torch.Tensor, *,
                max_len: int | None = None) -> Evicted:
    """Cuts every sequence to at most ``keep`` tokens: its last ``recent`` ones and, of the
    others, those of largest ``weights`` (ties: the earlier token; NaN below any number), chosen
    for each cached head by itself.  They are written in order to the pages of ``new_table``
    (int32 [sequences, pages], none of them a page that ``table`` names): later tokens are
    appended from place ``lens`` of the result on.  The old pages are the caller's again.

    ``weights``: fp32 [sequences, heads, tokens], at least ``max_len`` of them and as many as any
    sequence holds (tokens behind them would not count as held)."""
    kept, new_lens, new_weights = C.native().cache_evict(*cache, table, lens, weights, keep,
                                                         recent, new_table, max_len)
    return Evicted(kept, new_lens, new_weights)
