"""``token_logprobs`` against its definition in 64 bits: vocabularies from one
word to 151,936, several tokens a row, masked logits, ties, and its gradient.

Bounds.  A thread adds V / 256 terms at most, the block 13 more, each
exponential is off by its argument's rounding (|z - m| 2^-24 of itself) and two
units: the sum's relative error is under (V / 256 + 64 + 4 E|z - m|) 2^-24 =:
s 2^-24, E under the softmax.  ln s is off by as much; a log probability by
that and 4 roundings over |z| + |m| + |ln s|; the entropy by s 2^-24 over
1 + |ln s| + 2 E|z - m|; a gradient by (s + 4 |z - m|) 2^-24 over
p (|G| + |g_H| (|logp| + H)) + |g|, with |z - m| <= 140 where p is not 0.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check, directional

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def reference(x, tokens, k, temp, g_logp=None, g_ent=None, g_top=None):
    """Everything in 64 bits, with its bounds' magnitudes; x [T, V]."""
    T, V = x.shape
    z = x.detach().double() / temp
    live = (z > -INF).any(1)
    z[~live] = 0
    m = z.max(1, keepdim=True).values
    lns = torch.logsumexp(z - m, 1, keepdim=True)
    logp = z - m - lns
    p = logp.exp()
    spread = torch.where(p > 0, p * (z - m).abs(), torch.zeros_like(p)).sum(1, keepdim=True)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    H = -plogp.sum(1) * live
    s = V / 256 + 64 + 4 * spread                        # [T, 1]
    ok = (tokens >= 0) & (tokens < V)
    at = tokens.clamp(0, V - 1)
    dead = torch.full((), -INF, dtype=torch.float64, device=x.device)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    pick = lambda i: torch.where(live[:, None], logp.gather(1, i), dead)
    mag = lambda i: 4 * (z.gather(1, i).abs().clamp(max=1e30) + m.abs() + lns.abs()) + s
    order = torch.sort(x.detach().double(), dim=1, descending=True, stable=True).indices[:, :k]
    out = {"logprobs": (torch.where(ok, pick(at), zero), mag(at)),
           "entropy": (H, (s * (1 + lns.abs() + 2 * spread)).squeeze(1)),
           "top_tokens": order, "top_logprobs": (pick(order), mag(order))}
    if g_logp is not None or g_ent is not None or g_top is not None:
        gl = torch.zeros(T, tokens.shape[1], dtype=torch.float64, device=x.device) \
            if g_logp is None else torch.where(ok, g_logp.double(), zero)
        gt = torch.zeros(T, k, dtype=torch.float64, device=x.device) \
            if g_top is None else g_top.double()
        gh = torch.zeros(T, 1, dtype=torch.float64, device=x.device) \
            if g_ent is None else g_ent.double()[:, None]
        G = gl.sum(1, keepdim=True) + gt.sum(1, keepdim=True)
        dx = -p * G - gh * torch.where(p > 0, p * (logp + H[:, None]), zero)
        size = torch.where(p > 0, p * ((gl.abs().sum(1) + gt.abs().sum(1))[:, None]
                                       + gh.abs() * (logp.abs() + H[:, None])), zero)
        steps = s + 4 * (z - m).abs().clamp(max=140)
        size = size * steps
        for g, i in ((gl, at), (gt, order)):
            dx.scatter_add_(1, i, g)
            size.scatter_add_(1, i, 4 * g.abs())
        dx, size = dx * live[:, None] / temp, size / temp
        out["dx"] = (dx, size)
    return out


def run(x, tokens, k=0, temp=1.0, grads=True):
    T, V = x.shape
    x = x.detach().requires_grad_(grads)
    r = tt.token_logprobs(x, tokens, top_k=k, temperature=temp)
    g = torch.Generator(device=DEV).manual_seed(9)
    M = 0 if tokens is None else 1 if tokens.dim() == 1 else tokens.shape[1]
    tok2 = torch.zeros(T, 0, dtype=torch.int64, device=DEV) if tokens is None else \
        tokens.view(T, M).long()
    gl = torch.randn(T, M, generator=g, device=DEV)
    ge, gt = (torch.randn(*s, generator=g, device=DEV) for s in ((T,), (T, k)))
    w = reference(x, tok2, k, temp, *((gl, ge, gt) if grads else ()))
    assert r.entropy.dtype == r.logprobs.dtype == r.top_logprobs.dtype == F32
    if tokens is not None:
        assert r.logprobs.shape == tokens.shape
        check("logprobs", r.logprobs.detach().view(T, M), *w["logprobs"], 1)
    check("entropy", r.entropy.detach(), *w["entropy"], 1)
    assert torch.equal(r.top_tokens, w["top_tokens"])
    check("top_logprobs", r.top_logprobs.detach(), *w["top_logprobs"], 1)
    if grads:
        outs, gs = [r.entropy], [ge]
        if tokens is not None:
            outs, gs = outs + [r.logprobs], gs + [gl.view(tokens.shape)]
        if k:
            outs, gs = outs + [r.top_logprobs], gs + [gt]
        dx, = torch.autograd.grad(outs, [x], gs)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        check("dx", dx, *w["dx"], 1)
    return r


def logits(T, V, dtype, seed=0, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, V, generator=g, device=DEV) * scale
    x[torch.arange(T), torch.randint(0, V, (T,), generator=g, device=DEV)] += 6
    tok = torch.randint(0, V, (T, 3), generator=g, device=DEV)
    tok[::4, 1] = -100
    tok[1::4] = V
    return x.to(dtype), tok


@pytest.mark.parametrize("T,V,dtype,k,temp", [
    (1, 1, F32, 1, 1.0), (3, 2, BF, 2, 1.0), (47, 32000, F32, 8, 1.0), (5, 100, F16, 64, 0.7),
    (33, 1000, BF, 5, 1.0), (17, 1001, BF, 5, 1.3), (9, 4099, F16, 20, 1.0),
    (6, 151936, BF, 16, 1.0), (3, 151936, F32, 64, 0.5), (2, 151937, F16, 1, 1.0),
    (700, 257, BF, 3, 1.0), (900, 4097, BF, 64, 1.0), (500, 2050, F32, 33, 1.0), (40, 4104, F16, 64, 1.0), (1, 50000, BF, 10, 1.0), (2, 300000, BF, 7, 1.0),
    (300, 8192, BF, 4, 1.0), (64, 7, F32, 7, 2.0), (1500, 40000, BF, 16, 1.0),
    (1700, 20011, F16, 2, 1.0),
])
def test_both_directions(T, V, dtype, k, temp):
    x, tok = logits(T, V, dtype)
    run(x, tok, k, temp)


def test_tokens_forms():
    x, tok = logits(40, 500, BF)
    run(x, tok[:, 0])
    run(x, tok.int()[:, :1])
    run(x, None, 3)
    run(x, torch.empty(40, 0, dtype=torch.int64, device=DEV), 2)
    run(x, tok[:, :1].expand(40, 5).contiguous(), 2)          # the same token five times
    run(x, torch.randint(0, 500, (40, 100), device=DEV), 64)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("V", [130, 5000, 40000])
def test_masks(dtype, V):
    x, tok = logits(12, V, dtype)
    x[0, 1:] = -INF                       # one word left
    x[1] = -INF                           # none
    x[2, ::2] = torch.finfo(dtype).min    # the type's lowest value
    x[3] = torch.finfo(dtype).min         # everywhere: a uniform row
    x[4, 5:] = torch.finfo(dtype).min
    x[5, :V - 3] = -INF                   # the last three words
    x[6] = 0.25                           # all equal
    x[7, 100:] = -INF
    x[8] = 0.0
    x[8, ::3] = -0.0                      # equal to 0: the lowest index first
    tok[:, 0] = torch.tensor([0, 5, 1, 7, 2, V - 1, 9, 3, 4, 6, V, -1], device=DEV)
    run(x, tok, min(20, V))


def test_ties_and_orders_of_the_largest():
    V, k = 20000, 32
    x = torch.zeros(10, V, device=DEV, dtype=BF)
    x[0] = torch.arange(V, device=DEV).to(BF)                  # rising, many equal
    x[1] = -torch.arange(V, device=DEV).to(BF)                 # falling
    x[2] = (torch.arange(V, device=DEV) % 7).to(BF)            # few values
    x[3, ::2048] = 5                                           # far apart, all equal
    x[4, 4096:4096 + 200] = torch.linspace(1, 3, 200, device=DEV).to(BF)   # one run
    x[5, 8::2048] = torch.arange(10, device=DEV).to(BF)
    x[6, 0:V:64] = 1 + (torch.arange(0, V, 64, device=DEV) % 512).to(BF)   # a period
    x[7, :5] = 3
    x[8, -40:] = 2
    x[9, 12345] = -4
    tok = torch.randint(0, V, (10, 1), device=DEV)
    run(x, tok, k)
    run(x, tok, 64)
    # every large value in a few places of a long period
    y = torch.randn(4, 151936, device=DEV)
    y[:, ::2048] += 30
    y[:, 1::2048] += 30
    run(y.to(BF), tok[:4], 64)
    run(y, tok[:4], 64)


def test_nan_and_infinity():
    x, tok = logits(6, 3000, F32)
    plain = tt.token_logprobs(x, tok, top_k=4)
    x[1, 700] = float("nan")
    x[3, 2000] = INF
    r = tt.token_logprobs(x, tok, top_k=4)
    keep = [0, 2, 4, 5]
    for a, b in zip(r, plain):
        assert torch.equal(a[keep], b[keep])
    for row, at in ((1, 700), (3, 2000)):
        assert r.entropy[row].isnan() and r.top_tokens[row, 0] == at
        ok = (tok[row] >= 0) & (tok[row] < 3000)
        assert r.logprobs[row][ok].isnan().all() and (r.logprobs[row][~ok] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides(dtype):
    x, tok = logits(20, 1003, dtype)
    want = run(x, tok, 5)
    for width, lead in ((1024, 0), (1024, 8), (1100, 3), (2007, 1)):
        buf = torch.zeros(20, width, device=DEV, dtype=dtype)
        buf[:, lead:lead + 1003] = x
        got = run(buf[:, lead:lead + 1003], tok, 5)
        assert torch.equal(got.top_tokens, want.top_tokens)
    run(x.t().contiguous().t(), tok, 5)
    run(x[:1].expand(20, -1), tok, 5)
    run(x[::2], tok[::2], 5)


def test_offsets_over_32_bits():
    # 2^32 logits and more: the last rows' offsets pass 32 bits
    T, V = 16400, 262147
    x = torch.zeros(T, V, dtype=BF, device=DEV)
    rows = [0, 8191, 8192, 16398, 16399]
    g = torch.Generator(device=DEV).manual_seed(4)
    x[rows] = torch.randn(5, V, generator=g, device=DEV).to(BF)
    tok = torch.randint(0, V, (T, 1), generator=g, device=DEV)
    x.requires_grad_(True)
    r = tt.token_logprobs(x, tok, top_k=4)
    w = reference(x[rows], tok[rows], 4, 1.0, torch.ones(5, 1, device=DEV))
    check("logprobs", r.logprobs[rows].detach(), *w["logprobs"], 1)
    assert torch.equal(r.top_tokens[rows], w["top_tokens"])
    dx, = torch.autograd.grad(r.logprobs.sum(), [x])
    check("dx", dx[rows], *w["dx"], 1)


def test_gradients_of_some_outputs():
    x, tok = logits(30, 700, F32)
    x.requires_grad_(True)
    for name in ("logprobs", "entropy", "top_logprobs"):
        r = tt.token_logprobs(x, tok, top_k=6)
        o = getattr(r, name)
        g = torch.randn_like(o)
        dx, = torch.autograd.grad(o, [x], [g])
        kw = {"logprobs": "g_logp", "entropy": "g_ent", "top_logprobs": "g_top"}[name]
        check(name, dx, *reference(x, tok, 6, 1.0, **{kw: g})["dx"], 1)
    dx, = torch.autograd.grad(tt.token_logprobs(x, tok).logprobs.sum(), [x])   # an expanded 1
    check("sum", dx, *reference(x, tok, 0, 1.0, torch.ones_like(tok).float())["dx"], 1)


def test_gradients_by_differences():
    # third derivatives of log-softmax are under 1, so the central difference at
    # h = 1e-2 is off by under 1e-4 |d|^3 beside rounding: under 1e-2 of |grad|
    x, tok = logits(12, 64, F32, scale=1.0)
    gs = [torch.randn(12, 3, device=DEV), torch.randn(12, device=DEV)]
    f = lambda t: tt.token_logprobs(t, tok, temperature=1.2)[:2]
    x.requires_grad_(True)
    grads = torch.autograd.grad(f(x), [x], gs)
    directional(f, [x], gs, grads, 1e-2, 1e-2)


def test_same_result_twice_and_on_another_stream():
    x, tok = logits(200, 30000, BF)
    x.requires_grad_(True)

    def go():
        r = tt.token_logprobs(x, tok, top_k=9)
        dx, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), [x])
        return [*r, dx]
    a = go()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = go()
    s.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_no_rows():
    x = torch.zeros(0, 50, device=DEV, requires_grad=True)
    r = tt.token_logprobs(x, torch.zeros(0, 2, dtype=torch.int64, device=DEV), top_k=3)
    assert r.logprobs.shape == (0, 2) and r.top_tokens.shape == (0, 3)
    dx, = torch.autograd.grad(r.entropy.sum(), [x])
    assert dx.shape == (0, 50)


def test_refusals():
    x, tok = logits(4, 30, F32)
    f = tt.token_logprobs
    with pytest.raises(RuntimeError):
        f(x.cpu(), tok)
    with pytest.raises(RuntimeError):
        f(x, tok.cpu())
    with pytest.raises(TypeError):
        f(x.double(), tok)
    with pytest.raises(TypeError):
        f(x, tok.float())
    for a, kw in (((x[0], tok), {}), ((x, tok[:3]), {}), ((x, tok[None]), {}),
                  ((x[:, :0], tok), {}), ((x, tok), {"top_k": 31}), ((x, tok), {"top_k": -1}),
                  ((x, tok), {"temperature": 0.0}), ((x, tok), {"temperature": -1.0}),
                  ((x, tok), {"temperature": float("nan")}), ((x, tok), {"temperature": INF})):
        with pytest.raises(ValueError):
            f(*a, **kw)
    with pytest.raises(ValueError):
        f(torch.zeros(2, 100, device=DEV), None, top_k=65)


def test_differentiating_twice_is_refused():
    x, tok = logits(4, 30, F32)
    x.requires_grad_(True)
    g, = torch.autograd.grad(tt.token_logprobs(x, tok).entropy.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [x])


def test_logits_changed_in_place_are_noticed():
    x, tok = logits(4, 30, F32)
    x.requires_grad_(True)
    y = x * 1.0
    r = tt.token_logprobs(y, tok)
    y.detach().mul_(2.0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(r.entropy.sum(), [x])
