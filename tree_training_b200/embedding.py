"""Rows of an embedding table, scaled, with the table's gradient from sorted
tokens: one kernel forward; backward a stable sort of the tokens and one pass that
writes every row of the gradient once.  Every sum runs in a fixed order in fp32 (no
atomics), so two runs give the same bits.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _ops


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[ids]: ids [...] int64/int32, weight [V, H] fp32/bf16/fp16
    (any row stride, H up to 2^22) -> [..., H] of weight's type, rounded once.

    Differentiable in weight: a word's gradient is scale times the sum of its
    tokens' gradients in the order of the tokens, rounded once; ``padding_idx``
    (negative: from the end) gets none.  An id outside [0, V) gives a row of NaN
    and no gradient, and ``check_device_status`` raises.

    CUDA tensors only (no CPU path)."""
    return _ops.ext().embedding(ids, weight, float(scale), padding_idx)
