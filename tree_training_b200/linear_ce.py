"""The cross entropy of an LM head without its logits, by pieces of the vocabulary.

``ce.py`` gives one summed loss, by chunks of tokens whose logits a library product
forms.  Here the logits of a tile never leave the chip in the forward: the product's
epilogue reduces them to each row's maximum, sum of exponentials and labels' logits.
The backward forms them again a piece of the vocabulary at a time, so that the rows
of the weight's gradient are written once.

Which of the two: this one for losses token by token, several labels a token, a
gradient through lse, and in 16 bits in general (bf16, 2,560 wide, 151,936 words, with
gradients, one B200: 8,192 rows 19.3 ms and 1.2 GB against the chunks' 23.4 and 4.4, 47 rows
0.58 ms against 2.03).  ``ce.py`` for fp32 where one piece of a quarter of a gigabyte does
not hold the logits (4,096 rows of 32,000 words, 1,024 wide: 21.9 ms here, 17.7 there).

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
    after multiplication by a power of two that keeps them in range).  Workspaces are
    about rows * V / 8 bytes forward and the larger of 256 MB and rows * 8 KB backward.

    CUDA tensors only (no CPU path)."""
    return LinearCE(*_ops.ext().linear_cross_entropy(hidden, weight, labels, float(scale)))
