"""Log probabilities of given tokens with the entropy of their distributions and the likeliest
alternatives, and their gradient: how a packed model's answers are scored, and the loss of a
training step above packed layers.  No counterpart in the reference."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi as C

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # fp32 [...]
    entropy: torch.Tensor       # fp32 [...]
    top_logprobs: torch.Tensor  # fp32 [..., top]
    top_ids: torch.Tensor       # int64 [..., top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """For logits [..., vocab] (fp16, bf16 or fp32, on the GPU) and tokens [...] (int64 or int32):
    ``logits[token] - logsumexp(logits)``, ``-sum p log p`` and the ``top`` (at most 64) most
    likely tokens with their log probabilities, descending, equal ones by their number.

    A token outside the vocabulary (-100 for padding, say) is none: its logprob is 0.  Logits of
    -inf are tokens that cannot come up; a row of nothing else has logprobs of -inf and an entropy
    of 0.  The three floating results are differentiable in ``logits`` (once)."""
    return TokenLogprobs(*C.native().token_logprobs(logits, tokens, top))
