"""``token_logprobs`` at the ends of its range of temperatures: the definition's
limits, without NaN beside masked words, and an error outside the range."""
import math

import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
INF = float("inf")


@pytest.mark.parametrize("V", [100, 3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ends_of_the_range(V, dtype):
    x = torch.randn(5, V, device=DEV).to(dtype)
    x[1, V // 2:] = -INF
    x[2, ::2] = torch.finfo(dtype).min
    x[3] = -INF
    top = x.float().max(1).values
    x[0, 3], x[1, 4], x[2, 5], x[4, 6] = (float(t) + 1 for t in top[[0, 1, 2, 4]])
    tok = torch.tensor([3, 4, 5, 0, 6], device=DEV)
    x.requires_grad_(True)
    # cold: the largest word has probability 1
    r = tt.token_logprobs(x, tok, top_k=2, temperature=1e-20)
    live = [0, 1, 2, 4]
    assert (r.logprobs[live] == 0).all() and (r.entropy == 0).all()
    assert (r.top_tokens[live, 0] == tok[live]).all() and (r.top_logprobs[live, 1] < -1e15).all()
    assert (r.logprobs[3] == -INF).all()
    dx, = torch.autograd.grad(r.logprobs[live].sum() + r.entropy.sum(), [x])
    assert (dx == 0).all()
    # hot: all words are alike but those of the lowest value and -inf
    r = tt.token_logprobs(x, tok, temperature=1e20)
    words = (x > -1e30).sum(1).float()
    for v in (-r.logprobs[live], r.entropy[live]):
        assert ((v - words[live].log()).abs() < 1e-5 * math.log(V) + 1e-5).all()
    assert r.entropy[3] == 0 and r.logprobs[3] == -INF
    dx, = torch.autograd.grad(r.logprobs[live].sum(), [x])
    assert torch.isfinite(dx).all() and dx.abs().max() < 1e-19


def test_refusals():
    x, tok = torch.randn(4, 30, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for temp in (0.0, 1e-300, 1e-50, 1e-39, 9e-21, 1.1e20, 1e39, 1e300, INF, float("nan"), -1.0):
        with pytest.raises(ValueError):
            tt.token_logprobs(x, tok, temperature=temp)
