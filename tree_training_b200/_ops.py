"""What the op wrappers share: dtype codes, the current stream of a tensor's
device, and a call of the library with that device current."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

DTYPES = {torch.float32: _lib.TT_F32, torch.bfloat16: _lib.TT_BF16, torch.float16: _lib.TT_F16}

_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice
_functions: dict = {}


def call(device: torch.device, name: str, *args) -> None:
    """Calls the library on ``device``'s current stream (appended as the last
    argument); another current device is switched for the call."""
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(_lib.lib(), name)
    i = device.index
    if i == _current():
        rc = f(*args, _raw_stream(i))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _raw_stream(i))
    if rc:
        raise _lib.TTError(name, rc)


def once(backward):
    """A backward whose results carry no graph: differentiating them again is an
    error, as with ``once_differentiable``, whose cost only calls under
    ``create_graph`` pay here."""
    strict = once_differentiable(backward)

    def run(ctx, *grads):
        return strict(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def check_cuda(op: str, **tensors) -> torch.device:
    """Every given tensor (None is skipped) is on one CUDA device; returns it."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{op}: {name} must be a tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{op}: {name} must be a CUDA tensor (no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"{op}: {name} is on {t.device}, other tensors on {dev}")
    return dev


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def rows2d(t: torch.Tensor) -> torch.Tensor:
    """[rows, D] with unit last stride and non-overlapping rows (else a copy)."""
    if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()
