"""What the op wrappers share: dtype codes, the current stream of a tensor's
device, and a call of the library with that device current."""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.float32: _lib.TT_F32, torch.bfloat16: _lib.TT_BF16, torch.float16: _lib.TT_F16}

_raw_stream = torch._C._cuda_getCurrentRawStream


def stream_ptr(device: torch.device) -> int:
    return _raw_stream(device.index)


def call(device: torch.device, name: str, *args) -> None:
    """Calls the library on ``device``'s current stream (appended as the last
    argument); another current device is switched for the call."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _raw_stream(device.index))


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
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def rows2d(t: torch.Tensor) -> torch.Tensor:
    """[rows, D] with unit last stride and non-overlapping rows (else a copy)."""
    if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()
