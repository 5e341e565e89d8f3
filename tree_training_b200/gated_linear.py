"""The gated half of a decoder's feed-forward block: both projections, the
activation and their product in one kernel, with gradients.  (The way back,
``h @ w_down.T``, is a plain product.)
"""
from __future__ import annotations

import types
import weakref

import torch
from torch.nn.modules.module import _has_any_global_hook as has_any_global_hook
from torch.overrides import TorchFunctionMode

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
    of h under 1e-7 or so is lost there, as it is in fp16 itself.  Autocast does not
    change the types.

    CUDA tensors only (no CPU path)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation must be one of {sorted(ACTIVATIONS)}")
    return _ops.ext().gated_linear(x, w_gate, w_up, ACTIVATIONS[activation])


# Modules that are these activations and nothing else, by where they are defined: another
# class of the same name, or one derived from them, may do more.
_KNOWN = {
    "torch.nn.modules.activation": {"SiLU": "silu", "ReLU": "relu", "GELU": "gelu"},
    "transformers.activations": {"SiLUActivation": "silu", "GELUActivation": "gelu",
                                 "GELUTanh": "gelu_tanh", "PytorchGELUTanh": "gelu_tanh"},
}
_MULTIPLY = (torch.mul, torch.multiply, torch.Tensor.mul, torch.Tensor.multiply,
             torch.Tensor.__mul__, torch.Tensor.__rmul__)


def _activation_of(fn):
    """The name of a module's activation, None where it is not one of these."""
    cls = type(fn)
    name = _KNOWN.get(cls.__module__, {}).get(cls.__name__)
    if name is None or "forward" in fn.__dict__ or _has_hooks(fn):
        return None
    return "gelu_tanh" if cls is torch.nn.GELU and fn.approximate == "tanh" else name


class _Calls(TorchFunctionMode):
    """Every call that is made on tensors, but those inside the activation's module,
    which counts as one."""

    def __init__(self, act):
        super().__init__()
        self.calls, self.act, self.inside = [], act, False

    def __torch_function__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if not self.inside:
            self.note(func, args, kwargs, out)
        return out

    def note(self, func, args, kwargs, out):
        self.calls.append((func, args, kwargs, out, torch.is_grad_enabled(),
                           torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")))

    def enter(self, mod, args):
        self.inside = True

    def leave(self, mod, args, out):
        self.inside = False
        self.note(self.act, args, None, out)


def _is_plain(mod) -> bool:
    """Whether the module's forward is down(act(gate(x)) * up(x)) and nothing else, by
    the calls that it makes (a bound, dropout or a shape that is asked for is one more).
    Values show too little of it: a bound that they do not reach, zeros."""
    gate, up, down, act = mod.gate_proj, mod.up_proj, mod.down_proj, mod.act_fn
    x = torch.ones(2, gate.in_features, dtype=gate.weight.dtype, device=gate.weight.device)

    def plain(training, autocast) -> bool:
        mode = _Calls(act)
        hooks = [act.register_forward_pre_hook(mode.enter), act.register_forward_hook(mode.leave)]
        before = torch.is_autocast_enabled("cuda")
        context = [training, autocast, torch.get_autocast_dtype("cuda")]
        mod.training = training
        torch.set_autocast_enabled("cuda", autocast)
        try:
            with torch.set_grad_enabled(training), mode:
                result = mod.forward(x)
        except Exception:                     # (other arguments, say)
            return False
        finally:
            torch.set_autocast_enabled("cuda", before)
            if not before:
                torch.clear_autocast_cache()
            for hook in hooks:
                hook.remove()
        made = {}
        for func, args, kwargs, out, *within in mode.calls:
            if kwargs or within != context:
                return False
            if func is torch.nn.functional.linear and len(args) == 3:
                part = [p for p in (gate, up, down) if args[1] is p.weight and args[2] is p.bias]
            elif func is act and len(args) == 1:
                part = [act]
            elif func in _MULTIPLY and len(args) == 2:
                part = ["product"]
            else:
                return False
            if len(part) != 1 or part[0] in made:
                return False
            made[part[0]] = (args, out)
        if set(made) != {gate, up, down, act, "product"}:
            return False
        a, b = made["product"][0]
        if made[act][1] is not a:
            a, b = b, a
        return made[gate][0][0] is x and made[up][0][0] is x and made[act][0][0] is made[gate][1] \
            and a is made[act][1] and b is made[up][1] and made[down][0][0] is made["product"][1] \
            and result is made[down][1]
    training = mod.training
    devices = [x.device] if x.is_cuda else []
    try:
        with torch.random.fork_rng(devices=devices):
            # (one that sets autocast itself shows only where it changes it)
            return plain(True, False) and plain(False, False) and plain(True, True)
    finally:
        mod.training = training


def _has_hooks(mod) -> bool:
    return bool(mod._forward_hooks or mod._forward_pre_hooks or mod._backward_hooks
                or mod._backward_pre_hooks)


def _activation_of_parts(mod):
    """The activation's name where gate, up and activation are what the kernel computes
    (plain projections without bias, nothing attached to them), else None."""
    weights = []
    for part in (getattr(mod, "gate_proj", None), getattr(mod, "up_proj", None)):
        if type(part) is not torch.nn.Linear or part.bias is not None \
                or "forward" in part.__dict__ or _has_hooks(part) \
                or type(part.weight) not in (torch.nn.Parameter, torch.Tensor):
            return None
        weights.append(part.weight)
    act = getattr(mod, "act_fn", None)
    if weights[0].dtype != weights[1].dtype or weights[0].shape != weights[1].shape \
            or not isinstance(act, torch.nn.Module):
        return None
    return _activation_of(act)


# The forward of each class of which modules were taken.
_taken = weakref.WeakKeyDictionary()


def _gated_mlp_forward(self, *args, **kwargs):
    cls = type(self)
    name = _activation_of_parts(self)
    # what has changed since the module was taken goes by its own forward
    if name is None or kwargs or len(args) != 1 or _taken.get(cls, cls.forward) is not cls.forward \
            or has_any_global_hook():
        return cls.forward(self, *args, **kwargs)
    factors = [args[0], self.gate_proj.weight, self.up_proj.weight]
    kind = factors[0].device.type
    if torch.is_autocast_enabled(kind):       # (as the projections' own products)
        factors = [t.to(torch.get_autocast_dtype(kind)) for t in factors]
    return self.down_proj(gated_linear(*factors, name))


def fuse_gated_mlps(model) -> int:
    """Routes every gated feed-forward module of an HF model (``gate_proj``,
    ``up_proj`` and ``down_proj`` without biases, ``act_fn`` one of the activations)
    through :func:`gated_linear`.  Returns how many modules were patched; modules of
    another form or type keep their own forward, and so do those whose forward makes any
    other call on tensors (a bound, dropout, a branch on a shape; it is run to see them),
    sets autocast itself, has been replaced (by this function or another: wrap it after
    this call, as ``checkpoint_mlps`` does), or whose gate or up projection or activation
    has hooks.

    A patched module looks at its parts in every call: with an adapter in place of a
    projection, a hook on one or on the activation, or an activation that the kernel does
    not have, it goes by its class's forward for as long as that is so.  Under autocast it
    computes in autocast's type, as the projections would."""
    n = 0
    for mod in model.modules():
        name, down = _activation_of_parts(mod), getattr(mod, "down_proj", None)
        if name is None or type(down) is not torch.nn.Linear or "forward" in down.__dict__ \
                or getattr(mod.forward, "__func__", None) is not type(mod).forward \
                or mod.gate_proj.weight.dtype not in (torch.float32, torch.bfloat16,
                                                      torch.float16) \
                or any(c not in (mod.gate_proj, mod.up_proj, down, mod.act_fn)
                       for c in mod.children()) \
                or not _is_plain(mod):
            continue
        _taken[type(mod)] = type(mod).forward
        mod.forward = types.MethodType(_gated_mlp_forward, mod)
        n += 1
    return n
