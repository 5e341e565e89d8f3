"""Rotary positions for q and k in one kernel each way (``tt_rotary``): half and
interleaved pair layouts, all or part of the head, tables scaled for long
contexts.  Next to ``prologue.qk_norm_rope`` (q/k norm and a full-head turn in
the half layout) this serves layers without a q/k norm or with a partial turn.

The table is built once per model; the positions of a call are the tree's
depth-based position ids, so tokens of sibling branches share rows of it.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _ops

_SCALINGS = ("default", "linear", "dynamic", "yarn", "llama3", "longrope")


def _inverse_frequencies(dim: int, theta: float, scaling: dict, n_positions: int):
    """(frequencies [dim / 2] float64, factor of cos and sin)."""
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALINGS:
        raise ValueError(f"rotary_table: unknown scaling {kind!r}; one of {_SCALINGS}")
    exponent = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    freq = theta ** -exponent
    if kind == "default":
        return freq, 1.0
    factor = float(scaling.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError("rotary_table: the scaling factor must be at least 1")
    original = scaling.get("original_max_position_embeddings")
    if kind == "linear":
        return freq / factor, 1.0
    if original is None:
        raise ValueError(f"rotary_table: {kind} scaling needs original_max_position_embeddings")
    original = int(original)
    if kind == "dynamic":
        # the base grows with the length that is really used
        ratio = max(n_positions, original) / original
        base = theta * (factor * ratio - (factor - 1.0)) ** (dim / (dim - 2)) if dim > 2 else theta
        return base ** -exponent, 1.0
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = original * freq / (2.0 * math.pi)       # over the original context
        blend = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * (blend + (1.0 - blend) / factor), 1.0
    if kind == "longrope":
        per_dim = scaling["long_factor" if n_positions > original else "short_factor"]
        per_dim = torch.as_tensor(per_dim, dtype=torch.float64)
        if per_dim.numel() != dim // 2:
            raise ValueError("rotary_table: longrope needs one factor for each pair")
        stretch = float(scaling.get("factor", max(n_positions, original) / original))
        amp = scaling.get("attention_factor")
        if amp is None:
            amp = math.sqrt(1.0 + math.log(stretch) / math.log(original)) if stretch > 1.0 else 1.0
        return freq / per_dim, float(amp)
    # yarn: dims that turn more than beta_fast times over the original context
    # keep their frequency, those under beta_slow are divided by the factor,
    # with a ramp over the dim index between
    fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

    def index_of(turns):
        return dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    lo, hi = index_of(fast), index_of(slow)
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, dim - 1)
    if lo == hi:
        hi += 0.001
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / (hi - lo)).clamp(0.0, 1.0)
    amp = scaling.get("attention_factor")
    if amp is None:
        def m(scale):
            return 0.1 * scale * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        a, b = scaling.get("mscale"), scaling.get("mscale_all_dim")
        amp = m(a) / m(b) if a and b else m(1.0)
    return freq * (1.0 - ramp) + freq / factor * ramp, float(amp)


def rotary_table(n_positions: int, dim: int, theta: Optional[float] = None,
                 scaling: Optional[dict] = None, device=None) -> torch.Tensor:
    """fp32 [n_positions, dim]: dim / 2 cosines, then dim / 2 sines of each
    position.  ``scaling`` is a config's ``rope_scaling`` / ``rope_parameters``
    dict (default, linear, dynamic, yarn, llama3, longrope; ``dynamic`` and
    ``longrope`` go by ``n_positions``).  ``theta`` is the base; None: the
    ``rope_theta`` of ``scaling``, or 10,000.  Angles are formed in 64 bits: at
    position 40,000 a 32-bit angle is already off by 2e-3."""
    if n_positions < 1 or dim < 2 or dim % 2:
        raise ValueError("rotary_table: n_positions >= 1 and an even dim >= 2 required")
    scaling = dict(scaling or {})
    if theta is None:
        theta = scaling.get("rope_theta", 10000.0)
    freq, amp = _inverse_frequencies(dim, float(theta), scaling, int(n_positions))
    freq = freq.to(device=device)
    ang = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([ang.cos() * amp, ang.sin() * amp], 1).float()


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 table: torch.Tensor, interleaved: bool = False
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns the first R = table.shape[1] dims of every head of q [N, Hq, D] and
    k [N, Hk, D] (None: q alone) by the angles of ``positions`` [N]
    (int64/int32); the other dims pass through.  q and k share one of
    fp32/bf16/fp16 and may have any token and head strides (views of a packed
    projection, transposed views); results are contiguous.  Pairs are
    (i, i + R/2), or (2i, 2i + 1) with ``interleaved``.

    A position outside the table gives NaN in the turned dims and an error at
    the next ``check_device_status``.  Differentiable in q and k.  CUDA tensors
    only (no CPU path)."""
    return _ops.ext().apply_rotary(q, k, positions, table, bool(interleaved))
