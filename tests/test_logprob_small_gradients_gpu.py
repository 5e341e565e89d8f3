"""Gradients of ``token_logprobs`` far below the row's largest word, down to fp32's
subnormals, against 64 bits.

Bounds: with s = V / 256 + 64 + 4 E|z - m| (the sum's relative error in units of
2^-24), a gradient is off by (s + 4 |z - m|) 2^-24 over p (|G| + |g_H| (|logp| +
H)) + |g|, all over the temperature, and by half of the smallest subnormal: the
product of exponential and factor is rounded once.  |z - m| <= 170 where a
product with a factor under 2^64 is not 0.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("V", [300, 3000, 40000])
@pytest.mark.parametrize("temp", [2.0 ** -12, 0.0625, 1.0])
def test_small_gradients(V, temp):
    g = torch.Generator(device=DEV).manual_seed(5)
    T = 8
    x = torch.rand(T, V, generator=g, device=DEV) * -150 * temp
    x[:, 7] = 0.0
    x[3, ::2] = -float("inf")
    x[4, ::5] = torch.finfo(torch.float32).min
    tok = torch.randint(0, V, (T, 2), generator=g, device=DEV)
    gl, ge = torch.randn(T, 2, generator=g, device=DEV), torch.randn(T, generator=g, device=DEV)
    x.requires_grad_(True)
    r = tt.token_logprobs(x, tok, temperature=temp)
    dx, = torch.autograd.grad([r.logprobs, r.entropy], [x], [gl, ge])
    z = x.detach().double() / temp
    d = z - z.max(1, keepdim=True).values
    logp = d - torch.logsumexp(d, 1, keepdim=True)
    p = logp.exp()
    zero = torch.zeros_like(p)
    spread = torch.where(p > 0, p * d.abs(), zero).sum(1, keepdim=True)
    H = -torch.where(p > 0, p * logp, zero).sum(1, keepdim=True)
    glp, geh = gl.double(), ge.double()[:, None]
    want = -p * glp.sum(1, keepdim=True) - geh * torch.where(p > 0, p * (logp + H), zero)
    mag = torch.where(p > 0, p * (glp.abs().sum(1, keepdim=True) + geh.abs() * (logp.abs() + H)),
                      zero) * (V / 256 + 64 + 4 * spread + 4 * d.abs().clamp(max=170))
    want.scatter_add_(1, tok, glp)
    mag.scatter_add_(1, tok, 4 * glp.abs())
    assert (want.abs() / temp < 2.0 ** -130).any(), "no subnormal among them"
    check("dx", dx, want / temp, mag / temp, 1)
    masked = x.detach() == -float("inf")
    masked.scatter_(1, tok, False)
    assert (dx[masked] == 0).all()
