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

from . import _lib, _ops

MAX_EXPERTS = 1024
MAX_CHOICES = 64


class ExpertPlan:
    """``slots`` [T, k] int32: the sorted row of each choice, -1 if dropped;
    ``entries`` [T * k] int32: the choice (t * k + j) in each sorted row, -1
    past the kept ones; ``offsets`` [E + 1] int32: the first row of each
    expert, and the number of kept rows."""
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
    dev = _ops.check_cuda("expert_plan", expert_ids=expert_ids)
    if expert_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError("expert_plan: int64/int32 expert ids required")
    if expert_ids.dim() != 2:
        raise ValueError("expert_plan: expert_ids must be [T, k]")
    E = int(n_experts)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"expert_plan: n_experts must be in [1, {MAX_EXPERTS}]")
    T, k = expert_ids.shape
    if k > MAX_CHOICES:
        raise ValueError(f"expert_plan: at most {MAX_CHOICES} choices a token")
    n = T * k
    if n > 0x7fffffff:
        raise ValueError("expert_plan: more than 2^31 - 1 choices")
    ids = expert_ids.contiguous()
    ws = _lib.lib().tt_moe_plan_workspace_size(n, E)
    # one array for what a call writes; slots, entries, offsets, workspace
    buf = ids.new_empty(2 * n + E + 1 + ws // 4, dtype=torch.int32)
    slots, entries = buf[:n].view(T, k), buf[n:2 * n]
    offsets = buf[2 * n:2 * n + E + 1]
    p = buf.data_ptr()
    _ops.call(dev, "tt_moe_plan", ids.data_ptr(), ids.dtype == torch.int64, n, E, p, p + 4 * n,
              p + 8 * n, p + 4 * (2 * n + E + 1), ws)
    return ExpertPlan(slots, entries, offsets, T, k, E)


def _rows_op(name, src, plan, rows, *more):
    out = src.new_empty((rows, src.shape[1]))
    _ops.call(src.device, name, _ops.DTYPES[src.dtype], *more[:1], plan.n_tokens, plan.k,
              src.shape[1], plan.n_experts, plan.slots.data_ptr(), plan.offsets.data_ptr(),
              src.data_ptr(), *more[1:], out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _rows_op("tt_moe_dispatch", x, plan, plan.n_tokens * plan.k)

    @staticmethod
    @_ops.once
    def backward(ctx, dxs):
        return _rows_op("tt_moe_collect", dxs.contiguous(), ctx.plan, ctx.plan.n_tokens), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, plan):
        ctx.save_for_backward(ys, weights)
        ctx.plan = plan
        return _rows_op("tt_moe_combine", ys, plan, plan.n_tokens, _ops.DTYPES[weights.dtype],
                        weights.data_ptr())

    @staticmethod
    @_ops.once
    def backward(ctx, dy):
        ys, weights = ctx.saved_tensors
        plan = ctx.plan
        dy = dy.contiguous()
        dys, dw = torch.empty_like(ys), torch.empty_like(weights)
        _ops.call(ys.device, "tt_moe_spread", _ops.DTYPES[ys.dtype], _ops.DTYPES[weights.dtype],
                  plan.n_tokens, plan.k, ys.shape[1], plan.n_experts, plan.slots.data_ptr(),
                  plan.offsets.data_ptr(), dy.data_ptr(), ys.data_ptr(), weights.data_ptr(),
                  dys.data_ptr(), dw.data_ptr())
        return dys, dw, None


def _check_rows(op, name, t, rows, plan):
    _ops.check_cuda(op, **{name: t, "plan": plan.slots})
    if t.dtype not in _ops.DTYPES:
        raise TypeError(f"{op}: float32/bfloat16/float16 {name} required")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{op}: {name} must be [{rows}, H]")


def expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """xs [T * k, H] with xs[plan.slots[t, j]] = x[t]; rows past the kept ones
    are zero.  x [T, H] fp32/bf16/fp16; differentiable in x."""
    _check_rows("expert_dispatch", "x", x, plan.n_tokens, plan)
    x = x.contiguous()
    if _ops.wants_grad(x):
        return _Dispatch.apply(x, plan)
    return _rows_op("tt_moe_dispatch", x, plan, plan.n_tokens * plan.k)


def expert_combine(ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """y [T, H] = sum_j weights[t, j] * ys[plan.slots[t, j]] over the kept
    choices, in fp32, rounded once to ys's type.  ys [T * k, H] are the
    experts' outputs in sorted order, weights [T, k] fp32/bf16/fp16;
    differentiable in both (a dropped choice's weight gets gradient 0)."""
    _check_rows("expert_combine", "ys", ys, plan.n_tokens * plan.k, plan)
    _ops.check_cuda("expert_combine", ys=ys, weights=weights)
    if weights.dtype not in _ops.DTYPES:
        raise TypeError("expert_combine: float32/bfloat16/float16 weights required")
    if weights.shape != (plan.n_tokens, plan.k):
        raise ValueError(f"expert_combine: weights must be [{plan.n_tokens}, {plan.k}]")
    ys, weights = ys.contiguous(), weights.contiguous()
    if _ops.wants_grad(ys, weights):
        return _Combine.apply(ys, weights, plan)
    return _rows_op("tt_moe_combine", ys, plan, plan.n_tokens, _ops.DTYPES[weights.dtype],
                    weights.data_ptr())
