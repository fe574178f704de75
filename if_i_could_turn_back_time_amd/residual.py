"""The seam between two blocks of a decoder in one pass: the norm after a block, its gate and scale,
the residual stream, and the norm before the next block.  No counterpart in the reference."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi as C


class ResidualNorm(NamedTuple):
    stream: torch.Tensor  # x + scale * gate * branch (normalised first)
    normed: torch.Tensor  # the next block's input


def residual_norm(x: torch.Tensor, weight: torch.Tensor, branch: torch.Tensor | None = None, *,
                  gate: torch.Tensor | None = None, scale: float = 1.0,
                  branch_weight: torch.Tensor | None = None, eps: float = 1e-6) -> ResidualNorm:
    """With ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last dimension,

        b = rms(branch) * branch_weight        (the branch as it is without ``branch_weight``)
        stream = x + scale * gate * b          (x without a ``branch``, x itself)
        normed = rms(stream) * weight

    for x and branch [..., width] (fp16, bf16 or fp32, on the GPU), in fp32, both results rounded once
    (``normed`` is of the sum, not of its rounded value).  ``weight`` and ``branch_weight``: [width];
    ``gate``: [width], or x's shape, or that with leading dimensions of 1 from some one on ([sequences,
    1, width]: one for each sequence); all three of x's dtype or fp32.  A width of at most 32768.

    Differentiable (once) in all tensors.  Gradients that are sums over rows are summed in fp32 in a
    fixed order; what the gradient keeps is the inputs and two numbers a row."""
    return ResidualNorm(*C.native().residual_norm(x, weight, branch, gate, scale, branch_weight, eps))
