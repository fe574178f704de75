"""Embedding lookup with scaling and its gradient: the first layer of a model whose linear layers are
packed, trained beside them.  No counterpart in the reference."""
from __future__ import annotations

import torch

from . import _capi as C


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[tokens]`` for tokens [...] (int64 or int32) and weight [vocab, width] (fp16,
    bf16 or fp32, on the GPU): [..., width] of the weight's dtype, rounded once.

    A token outside the vocabulary (-100 for padding, say) is none: its row is 0 and it adds nothing to
    the gradient.  Differentiable in ``weight`` (once): the gradient is the whole table's, dense, each
    row the sum of its tokens' rows in fp32, rounded once, and the same from run to run."""
    return C.native().token_embedding(tokens, weight, scale)
