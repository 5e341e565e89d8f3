"""Log probabilities of given tokens, entropy and top alternatives of an LM
head's logits, with gradients: what a policy step on a trajectory tree takes
from the head (the leaf cross-entropy in ``ce.py`` gives one summed loss).

A token of a tree may have several successors: the last token of a node is
followed by the first token of each child.  ``tokens`` may therefore be
[rows, M], padded with any value outside the vocabulary, and a row's logits are
read once for all of them; :func:`tree_next_tokens` builds that array.

One kernel each way (``tt_token_logprobs_fwd/bwd``); sums and outputs are fp32
whatever the logits' type.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import _ops
from .packer import preorder_arrays

MAX_TOP_K = 64
IGNORE = -100


class TokenLogprobs(NamedTuple):
    """``logprobs`` has the shape of ``tokens``; ``entropy`` [rows];
    ``top_logprobs`` fp32 and ``top_tokens`` int64 [rows, top_k]."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def _forward(x, tokens, k, temperature, keep):
    T, V = x.shape
    M = tokens.shape[1]
    dev = x.device
    f32 = torch.float32
    logp = x.new_empty((T, M), dtype=f32)
    ent = x.new_empty(T, dtype=f32)
    top_lp = x.new_empty((T, k), dtype=f32)
    top_tok = tokens.new_empty((T, k))
    stats = x.new_empty((T, 4), dtype=f32) if keep else None
    _ops.call(dev, "tt_token_logprobs_fwd", _ops.DTYPES[x.dtype], T, V, x.data_ptr(),
              max(x.stride(0), V), tokens.data_ptr(), M, temperature, k, logp.data_ptr(),
              ent.data_ptr(), top_lp.data_ptr(), top_tok.data_ptr(),
              stats.data_ptr() if keep else None)
    return logp, ent, top_lp, top_tok, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, k: int, temperature: float):
        logp, ent, top_lp, top_tok, stats = _forward(x, tokens, k, temperature, True)
        ctx.save_for_backward(x, tokens, top_tok, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_tok)
        return logp, ent, top_lp, top_tok

    @staticmethod
    @_ops.once
    def backward(ctx, g_logp, g_ent, g_top, _):
        x, tokens, top_tok, stats = ctx.saved_tensors
        if g_logp is None and g_ent is None and g_top is None:
            return None, None, None, None
        T, V = x.shape
        g = [None if t is None else t.float().contiguous() for t in (g_logp, g_ent, g_top)]
        dx = torch.empty_like(x) if x.is_contiguous() else x.new_empty((T, V))
        _ops.call(x.device, "tt_token_logprobs_bwd", _ops.DTYPES[x.dtype], T, V, x.data_ptr(),
                  max(x.stride(0), V), tokens.data_ptr(), tokens.shape[1], ctx.temperature,
                  top_tok.shape[1], top_tok.data_ptr(),
                  *(None if t is None else t.data_ptr() for t in g), stats.data_ptr(),
                  dx.data_ptr())
        return dx, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities under softmax(logits / temperature).

    logits [rows, V] (fp32/bf16/fp16, any row stride); tokens [rows] or
    [rows, M] int64/int32, or None.  A token outside [0, V) is ignored: log
    probability 0, no gradient.  top_k <= min(64, V): the largest logits' tokens
    and log probabilities, the lowest index first among equals (NaN counts as
    the largest).  -inf logits have probability 0; a row of nothing but -inf
    has log probabilities -inf, entropy 0 and no gradient.

    Differentiable in ``logits`` through logprobs, entropy and top_logprobs.
    CUDA tensors only (no CPU path)."""
    dev = _ops.check_cuda("token_logprobs", logits=logits, tokens=tokens)
    if logits.dtype not in _ops.DTYPES:
        raise TypeError("token_logprobs: float32/bfloat16/float16 logits required")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("token_logprobs: logits must be [rows, V]")
    T, V = logits.shape
    k, temperature = int(top_k), float(temperature)
    if not 0 <= k <= min(MAX_TOP_K, V):
        raise ValueError(f"token_logprobs: top_k must be in [0, {min(MAX_TOP_K, V)}]")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("token_logprobs: temperature must be positive and finite")
    if tokens is None:
        tok = torch.empty((T, 0), dtype=torch.int64, device=dev)
    else:
        if tokens.dtype not in (torch.int64, torch.int32):
            raise TypeError("token_logprobs: int64/int32 tokens required")
        if tokens.dim() not in (1, 2) or tokens.shape[0] != T:
            raise ValueError("token_logprobs: tokens must be [rows] or [rows, M]")
        tok = tokens if tokens.dim() == 2 else tokens[:, None]
        tok = tok.to(torch.int64).contiguous()
    x = _ops.rows2d(logits)
    if _ops.wants_grad(logits):
        logp, ent, top_lp, top_tok = _TokenLogprobs.apply(x, tok, k, temperature)
    else:
        logp, ent, top_lp, top_tok, _ = _forward(x, tok, k, temperature, False)
    if tokens is not None and tokens.dim() == 1:
        logp = logp[:, 0]
    return TokenLogprobs(logp, ent, top_lp, top_tok)


def tree_next_tokens(roots: Sequence, ignore: int = IGNORE) -> np.ndarray:
    """The successors of every token of a forest in DFS order: int64 [N, M],
    M the most successors a token has (at least 1), padded with ``ignore``.
    Inside a node that is the next token; behind its last one, the first token
    of each child (of each grandchild behind an empty child)."""
    lens, parents, ids, _ = preorder_arrays(roots)
    n, N = len(lens), int(ids.shape[0])
    start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    after: list = [[] for _ in range(n)]        # first tokens below each node
    for c in range(n - 1, -1, -1):
        after[c].reverse()
        p = int(parents[c])
        if p >= 0:
            first = [int(ids[start[c]])] if lens[c] else list(after[c])
            after[p].extend(reversed(first))
    width = max([1] + [len(after[c]) for c in range(n) if lens[c]])
    out = np.full((N, width), ignore, np.int64)
    for c in range(n):
        b, e = int(start[c]), int(start[c + 1])
        if e > b:
            out[b:e - 1, 0] = ids[b + 1:e]
            out[e - 1, :len(after[c])] = after[c]
    return out
