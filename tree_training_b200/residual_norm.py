"""The edge between two blocks of a decoder layer: the norm after a block, its
gate, the residual sum and the norm before the next block, in place of the
layer's chain of elementwise ops (``gated_norm.py`` covers the norm inside a
delta-net block).  One kernel forward, two backward (``tt_residual_norm_fwd/bwd``):
the second adds up the column sums of the weights' gradients.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _ops

MAX_DIM = 16384


def residual_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, *,
                  post_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0, eps: float = 1e-6,
                  weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, r) with

        h = x, or RMSNorm(x) * (weight_offset + post_weight)
        r = residual + scale * gate * h
        y = RMSNorm(r) * (weight_offset + weight)

    x [..., D] (fp32/bf16/fp16, D <= 16384) is a block's output, ``residual``
    [..., D] the stream (x's type or fp32; None: zeros, for the first layer),
    y the next block's input and r the new stream, of the residual's type.
    y is formed from r before its rounding.  ``gate`` has x's type: [D] one
    value a channel, [..., 1] one a row, [..., D] one an element.  weight and
    post_weight [D] are fp32 or of x's type.  ``weight_offset`` 1 serves norms
    whose weights are kept around zero.

    Differentiable in x, residual, weight, post_weight and gate.  CUDA tensors
    only (no CPU path)."""
    return _ops.ext().residual_norm(x, residual, weight, post_weight, gate, float(scale),
                                    float(eps), float(weight_offset), MAX_DIM)
