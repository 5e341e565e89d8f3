"""Loads the torch bindings of the layer operators (``csrc/torch/tt_torch.cpp``:
argument checks, outputs and autograd nodes around the C ABI)."""
from __future__ import annotations

from . import _lib

_ext = None


def ext():
    """The bindings; there is no fallback if they are missing."""
    global _ext
    if _ext is None:
        _lib.lib()          # the C ABI they call; raises if it is missing
        try:
            from . import _tt_torch
        except ImportError as e:
            raise RuntimeError("the torch bindings are missing: build them with "
                               "`python -m tree_training_b200.build` (there is no fallback)") from e
        _ext = _tt_torch
    return _ext
