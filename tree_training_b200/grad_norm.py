"""The norm of all gradients together, and gradients scaled to a largest norm: two
launches for hundreds of tensors, without waiting for the device.
"""
from __future__ import annotations

from typing import Iterable, Optional, Sequence

import torch

from . import _ops


def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``tensors`` (fp32/bf16/fp16, mixed, on one
    device) together: fp32, one element, on their device.  norm_type 1, 2 or inf.
    Sums are formed in 64 bits across packs of 16 bytes and in a fixed order; NaN
    and infinities come through."""
    return _ops.ext().grad_norm(list(tensors), float(norm_type))


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                   eps: float = 1e-6, norm: Optional[torch.Tensor] = None,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Multiplies every gradient by min(1, max_norm / (norm + eps)) and returns the
    norm (of before).

    In place, or into ``out`` (one tensor for each gradient, of its shape, type and
    strides; it may be the gradient itself).  ``norm`` [1 element, fp32, on the
    device, no part of what is written]: go by this norm (one summed over ranks, say)
    instead of computing it.
    Where the norm is not finite the factor is 0 or NaN, as the formula gives it.

    Tensors that are written must fill their memory without gaps, and none may share
    memory with another.  CUDA tensors only (no CPU path)."""
    return _ops.ext().clip_grad_norm(list(grads), float(max_norm), float(norm_type), float(eps),
                                     norm, None if out is None else list(out))
