"""``token_logprobs`` on rows whose words all have the type's lowest (or highest)
value, at temperatures around 1 and small ones, against 64 bits.

Bounds.  A log probability is (x - m) / temperature - ln s: three roundings over
|z - m| and |ln s|, one of the temperature's exponent factor, and ln s is off by
the sum's relative error, under (V / 256 + 64 + 4 E|z - m|) 2^-24 =: s 2^-24
(a thread adds V / 256 terms at most).  The largest values themselves do not
enter.  An entropy is off by s 2^-24 over 1 + |ln s| + 2 E|z - m|, a gradient by
(s + 4 |z - m|) 2^-24 over p |G| + |g|, with |z - m| <= 140 where p is not 0.
A log probability under fp32's range is -inf.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def rows(T, V, dtype):
    lowest, highest = torch.finfo(dtype).min, torch.finfo(dtype).max
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(T, V, generator=g, device=DEV).to(dtype)
    x[0] = lowest                          # a mask that leaves nothing
    x[1] = lowest
    x[1, ::3] = -INF
    x[2] = -INF                            # one word, of the lowest value
    x[2, V // 2] = lowest
    x[3] = lowest                          # one word left
    x[3, V // 3] = 1.5
    x[4] = highest
    x[5] += 20                             # x / temperature large, differences small
    x[6] = lowest
    x[6, 1::2] = lowest / 2
    tok = torch.randint(0, V, (T, 3), generator=g, device=DEV)
    tok[:7, 0] = torch.tensor([V - 1, 1, V // 2, V // 3, 7, 3, 1], device=DEV)
    tok[7::5, 1] = -1
    return x, tok


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("T,V,k", [
    (12, 130, 0), (12, 130, 20), (1100, 130, 20), (1030, 900, 5), (12, 3000, 16),
    (12, 3000, 20), (12, 40000, 0), (12, 40000, 20), (300, 70000, 8),
])
@pytest.mark.parametrize("temp", [0.0625, 0.75, 1.0, 1.25])
def test_rows_of_the_lowest_value(T, V, k, dtype, temp):
    # (temperatures that fp32 holds exactly)
    x, tok = rows(T, V, dtype)
    x.requires_grad_(True)
    r = tt.token_logprobs(x, tok, top_k=k, temperature=temp)
    g = torch.randn(T, 3, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    dx, = torch.autograd.grad(r.logprobs, [x], [g])

    z = x.detach().double() / temp
    d = z - z.max(1, keepdim=True).values
    lns = torch.logsumexp(d, 1, keepdim=True)
    logp = d - lns
    p = logp.exp()
    spread = torch.where(p > 0, p * d.abs(), torch.zeros_like(p)).sum(1, keepdim=True)
    s = V / 256 + 64 + 4 * spread
    ok = tok >= 0
    at = tok.clamp(min=0)
    in_range = lambda t: torch.where(t < torch.finfo(F32).min, torch.full_like(t, -INF), t)
    # (d is -inf where the result is: its size does not matter there)
    size = lambda i: (4 * (d.gather(1, i).abs().clamp(max=1e38) + lns.abs()) + s)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    check("logprobs", r.logprobs.detach(), torch.where(ok, in_range(logp.gather(1, at)), zero),
          size(at), 1)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    check("entropy", r.entropy.detach(), -plogp.sum(1),
          (s * (1 + lns.abs() + 2 * spread)).squeeze(1), 1)
    order = torch.sort(x.detach().double(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.top_tokens, order)
    check("top_logprobs", r.top_logprobs.detach(), in_range(logp.gather(1, order)), size(order), 1)
    gl = torch.where(ok, g.double(), zero)
    want = -p * gl.sum(1, keepdim=True)
    mag = p * gl.abs().sum(1, keepdim=True) * (s + 4 * d.abs().clamp(max=140))
    want.scatter_add_(1, at, gl)
    mag.scatter_add_(1, at, 4 * gl.abs())
    check("dx", dx, want / temp, mag / temp, 1)


def test_the_uniform_row_has_minus_log_of_its_words():
    for dtype in (F32, BF):
        x = torch.full((3, 1000), torch.finfo(dtype).min, dtype=dtype, device=DEV)
        for temp in (0.7, 1.0, 1.3):
            r = tt.token_logprobs(x, torch.arange(3, device=DEV), top_k=2, temperature=temp)
            for v in (r.logprobs, r.top_logprobs, -r.entropy):
                assert ((v + 6.907755278982137).abs() < 1e-5).all()
