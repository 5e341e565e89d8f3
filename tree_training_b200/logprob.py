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


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities under softmax(logits / temperature), the temperature in
    [1e-20, 1e20].

    logits [rows, V] (fp32/bf16/fp16, any row stride); tokens [rows] or
    [rows, M] int64/int32, or None.  A token outside [0, V) is ignored: log
    probability 0, no gradient.  top_k <= min(64, V): the largest logits' tokens
    and log probabilities, the lowest index first among equals (NaN counts as
    the largest).  -inf logits have probability 0; a row of nothing but -inf
    has log probabilities -inf, entropy 0 and no gradient.

    The gradient's time at the given tokens grows with M times the row's different
    tokens: made for the successors in a tree, not for whole vocabularies.

    Differentiable in ``logits`` through logprobs, entropy and top_logprobs.
    CUDA tensors only (no CPU path)."""
    return TokenLogprobs(*_ops.ext().token_logprobs(logits, tokens, int(top_k),
                                                    float(temperature), MAX_TOP_K))


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
