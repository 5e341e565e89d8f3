"""Tokens sorted by expert and back, with the router's weights, and gradients:
what stands on either side of the experts' products in a mixture layer.

``expert_plan`` sorts the router's choices once; ``expert_dispatch`` lays the
tokens out expert by expert (expert e's rows are [offsets[e], offsets[e + 1]))
and ``expert_combine`` brings the experts' outputs back as one weighted sum a
token.  No call waits for the device: the number of kept rows stays there, and
the sorted arrays always have n_tokens * k rows, zero past the kept ones.
Every sum runs in a fixed order in fp32 (no atomics).
"""
from __future__ import annotations

import torch

from . import _ops

MAX_EXPERTS = 1024
MAX_CHOICES = 64


class ExpertPlan:
    """``slots`` [T, k] int32: the sorted row of each choice, -1 if dropped;
    ``entries`` [T * k] int32: the choice (t * k + j) in each sorted row, -1
    past the kept ones; ``offsets`` [E + 1] int32: the first row of each
    expert, and the number of kept rows.

    A plan may be made or changed by the caller: a slot outside the T * k rows
    drops its choice; rows below offsets[E] that no slot names are not written."""
    __slots__ = ("slots", "entries", "offsets", "n_tokens", "k", "n_experts")

    def __init__(self, slots, entries, offsets, n_tokens, k, n_experts):
        self.slots, self.entries, self.offsets = slots, entries, offsets
        self.n_tokens, self.k, self.n_experts = n_tokens, k, n_experts

    @property
    def counts(self) -> torch.Tensor:
        """Rows of each expert [E]."""
        return self.offsets[1:] - self.offsets[:-1]


def expert_plan(expert_ids: torch.Tensor, n_experts: int) -> ExpertPlan:
    """Sorts the choices ``expert_ids`` [T, k] (int64/int32) by expert, each
    expert's in token order.  An id outside [0, n_experts) drops the choice.
    k <= 64, n_experts <= 1024.  CUDA tensors only (no CPU path)."""
    slots, entries, offsets = _ops.ext().expert_plan(expert_ids, int(n_experts), MAX_EXPERTS,
                                                     MAX_CHOICES)
    return ExpertPlan(slots, entries, offsets, *slots.shape, int(n_experts))


def expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """xs [T * k, H] with xs[plan.slots[t, j]] = x[t]; rows past the kept ones
    are zero.  x [T, H] fp32/bf16/fp16; differentiable in x."""
    return _ops.ext().expert_dispatch(x, plan.slots, plan.offsets)


def expert_combine(ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """y [T, H] = sum_j weights[t, j] * ys[plan.slots[t, j]] over the kept
    choices, in fp32, rounded once to ys's type.  ys [T * k, H] are the
    experts' outputs in sorted order, weights [T, k] fp32/bf16/fp16;
    differentiable in both (a dropped choice's weight gets gradient 0)."""
    return _ops.ext().expert_combine(ys, weights, plan.slots, plan.offsets)
