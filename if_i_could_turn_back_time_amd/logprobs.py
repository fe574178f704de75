"""Log probabilities of given tokens with the entropy of their distributions and the likeliest
alternatives, and their gradient: how a packed model's answers are scored, and the loss of a
training step above packed layers, from logits or, without their being kept, from the hidden states
under the head.  No counterpart in the reference."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi as C
from .linear import PackedWeight, QuantLinear, _kernel_input

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


class HeadLogprobs(NamedTuple):
    logprob: torch.Tensor  # fp32 [...]
    entropy: torch.Tensor  # fp32 [...]


def head_logprobs(hidden: torch.Tensor, head, tokens: torch.Tensor) -> HeadLogprobs:
    """``token_logprobs(hidden @ W.T, tokens)`` without the logits: they are reduced where they are
    summed, in fp32, and computed again for the gradient, a piece at a time.

    ``head``: a weight [vocab, width] (fp16 or bf16, as ``hidden`` [..., width]), differentiable (once)
    as ``hidden`` is; or a ``QuantLinear`` without a bias or a ``PackedWeight``, which are frozen: then
    ``hidden`` is cast as ``packed_linear`` does (and may be fp32).  Tokens as for
    :func:`token_logprobs`: one outside the vocabulary is none, and its row gets no gradient but its
    entropy's, nor gives the weight any, whatever ``hidden`` holds there.

    The gradients' products take each logit's gradient in 16 bits, as a backward pass through 16-bit
    logits does, but for the given token's, whose rounding is made up for: gradients of log probabilities
    are as near as their own rounding lets them be where no other token is likely, gradients of entropies
    1.4 times as far off (``token_logprobs`` of fp32 logits keeps more).  (A packed head takes them in
    fp32 under fp32 ``hidden``, and where it is rotated or its scales leave 16 bits.)"""
    if isinstance(head, (QuantLinear, PackedWeight)):
        if isinstance(head, QuantLinear):
            if head.bias is not None:
                raise ValueError("head_logprobs takes a head without a bias; with one: "
                                 "token_logprobs(head(hidden), tokens)")
            n, k, fmt, f16_exact = head.out_features, head.in_features, head.fmt, head._f16_exact
            bf16_exact = f16_exact if head._bf16_exact is None else head._bf16_exact
            if head.range_check and hidden.dim() and hidden.shape[-1] == k:
                _kernel_input(hidden.detach().reshape(-1, k), k, fmt, head.fwht_block, True, f16_exact)
        else:
            n, k, fmt, f16_exact = head.N, head.K, head.fmt_name, head.f16_exact
            bf16_exact = f16_exact  # a range within bf16's
        r = C.native().packed_head_logprobs(hidden, head.wdev, tokens, n, k, C.FMT_BY_NAME[fmt],
                                            head.fwht_block, f16_exact, bf16_exact)
    else:
        r = C.native().head_logprobs(hidden, head, tokens)
    return HeadLogprobs(*r)
