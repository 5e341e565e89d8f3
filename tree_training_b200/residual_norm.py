"""The edge between two blocks of a decoder layer in one kernel each way
(``tt_residual_norm_fwd/bwd``): the norm after a block, its gate, the residual
sum and the norm before the next block, in place of the layer's chain of
elementwise ops (``gated_norm.py`` covers the norm inside a delta-net block).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, _ops
from .attention import _status_word

MAX_DIM = 16384
_NONE, _CHANNEL, _ROW, _FULL = 0, 1, 2, 3


def _ptr(t):
    return None if t is None else t.data_ptr()


def _new(x, dtype):
    """A contiguous array of x's shape (``empty_like`` keeps an x that is dense in
    another order as it is)."""
    if dtype == x.dtype and x.is_contiguous():
        return torch.empty_like(x)
    return x.new_empty(x.shape, dtype=dtype)


def _forward(x, res, w, post, gate, mode, scale, eps, offset, keep):
    T, D = x.shape
    rt = x.dtype if res is None else res.dtype
    y = _new(x, x.dtype)
    r = _new(x, rt)
    stats = x.new_empty((T, 2), dtype=torch.float32) if keep else None
    _ops.call(x.device, "tt_residual_norm_fwd", _ops.DTYPES[x.dtype], _ops.DTYPES[rt], T, D,
              x.data_ptr(), x.stride(0), _ptr(res), 0 if res is None else res.stride(0),
              w.data_ptr(), _ptr(post), w.dtype == torch.float32, offset, _ptr(gate),
              0 if gate is None else gate.stride(0), mode, scale, eps, y.data_ptr(),
              r.data_ptr(), _ptr(stats), _status_word(x.device).data_ptr())
    return y, r, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w, post, gate, mode: int, scale: float, eps: float, offset: float):
        y, r, stats = _forward(x, res, w, post, gate, mode, scale, eps, offset, True)
        ctx.save_for_backward(x, res, w, post, gate, stats)
        ctx.args = (mode, scale, offset)
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @_ops.once
    def backward(ctx, dy, dr):
        x, res, w, post, gate, stats = ctx.saved_tensors
        mode, scale, offset = ctx.args
        if dy is None and dr is None:
            return (None,) * 9
        T, D = x.shape
        dev, rt = x.device, x.dtype if res is None else res.dtype
        need = ctx.needs_input_grad
        # the same array where nothing stands between the two
        same = post is None and mode == _NONE and scale == 1.0 and rt == x.dtype
        new = torch.empty_like if T else torch.zeros_like
        dres = _new(x, rt) if need[1] or (same and need[0]) else None
        dx = _new(x, x.dtype) if need[0] and not same else None
        dw = new(w) if need[2] else None
        dpost = new(post) if need[3] else None
        dgate = None
        if need[4]:
            dgate = new(gate) if mode == _CHANNEL else gate.new_empty(gate.shape)
        dy = None if dy is None else _ops.rows2d(dy)
        dr = None if dr is None else _ops.rows2d(dr)
        blocks = _lib.lib().tt_residual_norm_bwd_blocks(T, D)
        part = x.new_empty(3 * blocks * D, dtype=torch.float32)
        _ops.call(dev, "tt_residual_norm_bwd", _ops.DTYPES[x.dtype], _ops.DTYPES[rt], T, D,
                  x.data_ptr(), x.stride(0), _ptr(res), 0 if res is None else res.stride(0),
                  w.data_ptr(), _ptr(post), w.dtype == torch.float32, offset, _ptr(gate),
                  0 if gate is None else gate.stride(0), mode, scale, stats.data_ptr(),
                  _ptr(dy), 0 if dy is None else dy.stride(0), _ptr(dr),
                  0 if dr is None else dr.stride(0), _ptr(dx), _ptr(dres), _ptr(dgate), _ptr(dw),
                  _ptr(dpost), part.data_ptr(), blocks, _status_word(dev).data_ptr())
        if same and need[0]:
            dx = dres
        return dx, dres if need[1] else None, dw, dpost, dgate, None, None, None, None


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
    dev = _ops.check_cuda("residual_norm", x=x, residual=residual, weight=weight,
                          post_weight=post_weight, gate=gate)
    if x.dtype not in _ops.DTYPES:
        raise TypeError("residual_norm: float32/bfloat16/float16 x required")
    if residual is not None and residual.dtype not in (x.dtype, torch.float32):
        raise TypeError("residual_norm: residual must have x's type or float32")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError(f"residual_norm: x must be [..., D] with 1 <= D <= {MAX_DIM}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError("residual_norm: residual must have x's shape")
    D = x.shape[-1]
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is None:
            continue
        if w.shape != (D,):
            raise ValueError(f"residual_norm: {name} must be [{D}]")
        if w.dtype not in (x.dtype, torch.float32) or w.dtype != weight.dtype:
            raise TypeError(f"residual_norm: {name} must be float32 or x's type, like weight")
    mode = _NONE
    if gate is not None:
        if gate.dtype != x.dtype:
            raise TypeError("residual_norm: gate must have x's type")
        if gate.shape == (D,) and (x.dim() > 1 or D > 1):
            mode = _CHANNEL
        elif gate.shape == x.shape:
            mode = _FULL
        elif gate.shape == x.shape[:-1] + (1,):
            mode = _ROW
        else:
            raise ValueError("residual_norm: gate must be [D], [..., 1] or [..., D]")
    shape = x.shape
    two = x.dim() == 2
    x2 = _ops.rows2d(x if two else x.reshape(-1, D))
    r2 = None if residual is None else _ops.rows2d(residual if two else residual.reshape(-1, D))
    if mode == _CHANNEL:
        g2 = gate.contiguous()
    elif mode == _NONE:
        g2 = None
    else:
        g2 = _ops.rows2d(gate if two else gate.reshape(-1, gate.shape[-1]))
    w2 = weight.contiguous()
    p2 = None if post_weight is None else post_weight.contiguous()
    args = (x2, r2, w2, p2, g2, mode, float(scale), float(eps), float(weight_offset))
    if _ops.wants_grad(x, residual, weight, post_weight, gate):
        y, r = _ResidualNorm.apply(*args)
    else:
        y, r, _ = _forward(*args, False)
    return (y, r) if two else (y.view(shape), r.view(shape))
