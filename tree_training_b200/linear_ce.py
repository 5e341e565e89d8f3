"""The cross entropy of an LM head without its logits, by pieces of the vocabulary.

``ce.py`` gives one summed loss, by chunks of tokens whose logits a library product
forms.  Here the logits of a tile never leave the chip in the forward: the product's
epilogue reduces them to each row's maximum, sum of exponentials and labels' logits.
The backward forms them again a piece of the vocabulary at a time, so that the rows
of the weight's gradient are written once.

As in ``logprob.py`` a token of a tree may have several successors: labels may be
[rows, M], padded with any value outside the vocabulary (``tree_next_tokens``).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ops


class LinearCE(NamedTuple):
    """``losses`` fp32 with the shape of the labels, ``lse`` fp32 [rows]."""
    losses: torch.Tensor
    lse: torch.Tensor


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         scale: float = 1.0) -> LinearCE:
    """With z = scale * hidden @ weight.T:  lse = logsumexp(z),
    losses[t, m] = lse[t] - z[t, labels[t, m]].

    hidden [rows, H] and weight [V, H] of one type (fp32/bf16/fp16, any row
    strides; 16-bit rows that do not start on 16-byte boundaries are copied first);
    labels [rows] or [rows, M] int64/int32.  A label outside [0, V) is ignored: loss
    0, no gradient.  Sums are fp32.  An infinite logit gives NaN.

    Differentiable in hidden and weight through losses and lse; the logits'
    gradients are rounded to hidden's type once, for the products that follow (fp16:
    after multiplication by a power of two that keeps them in range).

    CUDA tensors only (no CPU path)."""
    return LinearCE(*_ops.ext().linear_cross_entropy(hidden, weight, labels, float(scale)))
