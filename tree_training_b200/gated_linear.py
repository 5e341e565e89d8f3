"""The gated half of a decoder's feed-forward block: both projections, the
activation and their product in one kernel, with gradients.  (The way back,
``h @ w_down.T``, is a plain product.)
"""
from __future__ import annotations

import types

import torch

from . import _ops

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 activation: str = "silu") -> torch.Tensor:
    """h = activation(x @ w_gate.T) * (x @ w_up.T)

    x [..., H], w_gate and w_up [F, H] of one type (fp32/bf16/fp16), F below 2^30 - 255
    -> [..., F]; activation one of silu, gelu, gelu_tanh, relu.  Sums are fp32, h is rounded
    once.  Any row strides; 16-bit rows that do not start on 16-byte boundaries are
    copied first.  The two weights may be halves of one tensor.

    Differentiable in all three.  For the backward the two products are kept in
    fp32 (8 bytes an element of h); their gradients are rounded to x's type once,
    for the products that give dx and the weights' gradients: in fp16 a gradient
    of h under 1e-7 or so is lost there, as it is in fp16 itself.

    CUDA tensors only (no CPU path)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation must be one of {sorted(ACTIVATIONS)}")
    return _ops.ext().gated_linear(x, w_gate, w_up, ACTIVATIONS[activation])


def _activation_of(fn):
    """The name of a module's activation, None where it is not one of these."""
    if isinstance(fn, torch.nn.GELU):
        return "gelu_tanh" if fn.approximate == "tanh" else "gelu"
    return {"SiLU": "silu", "SiLUActivation": "silu", "ReLU": "relu", "GELUActivation": "gelu",
            "GELUTanh": "gelu_tanh", "PytorchGELUTanh": "gelu_tanh"}.get(type(fn).__name__)


@torch.no_grad()
def _is_plain(mod) -> bool:
    """Whether the module's forward is down(act(gate(x)) * up(x)) and nothing else
    (no dropout, sparsity or clamp), by what it gives for a few rows in training."""
    w = mod.gate_proj.weight
    x = torch.linspace(-3, 3, 4 * w.shape[1], dtype=torch.float32).view(4, -1).sin()
    x = x.to(w.device, w.dtype)
    training = mod.training
    mod.training = True
    try:
        with torch.random.fork_rng(devices=[w.device] if w.is_cuda else []):
            y = mod.forward(x)
    finally:
        mod.training = training
    want = mod.down_proj(mod.act_fn(mod.gate_proj(x)) * mod.up_proj(x))
    return isinstance(y, torch.Tensor) and y.shape == want.shape and \
        torch.allclose(y.float(), want.float(), rtol=2e-2, atol=1e-3 * float(want.abs().max()))


def _has_hooks(mod) -> bool:
    return any(getattr(mod, a) for a in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks",
                                         "_backward_pre_hooks"))


def _gated_mlp_forward(self, x):
    return self.down_proj(gated_linear(x, self.gate_proj.weight, self.up_proj.weight,
                                       self._tt_activation))


def fuse_gated_mlps(model) -> int:
    """Routes every gated feed-forward module of an HF model (``gate_proj``,
    ``up_proj`` and ``down_proj`` without biases, ``act_fn`` one of the activations)
    through :func:`gated_linear`.  Returns how many modules were patched; modules of
    another form or type keep their own forward, and so do those whose forward does
    more than that, has been replaced (by this function or another: wrap it after
    this call, as ``checkpoint_mlps`` does), or whose gate or up projection has hooks."""
    n = 0
    for mod in model.modules():
        parts = [getattr(mod, a, None) for a in ("gate_proj", "up_proj", "down_proj")]
        if not all(type(p) is torch.nn.Linear for p in parts) or not hasattr(mod, "act_fn") \
                or getattr(mod.forward, "__func__", None) is not type(mod).forward \
                or _has_hooks(parts[0]) or _has_hooks(parts[1]):
            continue
        if parts[0].weight.dtype not in (torch.float32, torch.bfloat16, torch.float16) or \
                any(c not in (*parts, mod.act_fn) for c in mod.children()):
            continue
        name = _activation_of(mod.act_fn)
        if name is None or parts[0].bias is not None or parts[1].bias is not None \
                or not _is_plain(mod):
            continue
        mod._tt_activation = name
        mod.forward = types.MethodType(_gated_mlp_forward, mod)
        n += 1
    return n
