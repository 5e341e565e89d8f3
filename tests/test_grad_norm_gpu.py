"""The norm of many tensors and their scaling against the formulas in 64 bits."""
import math

import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import EPS, UNIT

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


def norm_of(ts, p):
    return torch.linalg.vector_norm(torch.cat([t.double().reshape(-1) for t in ts]), p)


def make(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * scale).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def close(norm, want, adds=16):
    """A pack's 8 values go through 8 fp32 roundings (in a root: half of that), the
    result through one."""
    assert norm.dtype == F32 and norm.shape == ()
    assert abs(float(norm) - float(want)) <= adds * EPS * float(want), (float(norm), float(want))


def scaled(got, t, norm, max_norm, eps=1e-6):
    """got = t * min(1, max_norm / (norm + eps)): the fp32 factor's roundings (three,
    and the norm's), the product's, and the result's own."""
    c = min(1.0, max_norm / (float(norm) + eps))
    want = t.double() * c
    bound = UNIT[t.dtype] * want.abs() + 24 * EPS * want.abs() + \
        {F32: 2.0 ** -149, BF: 2.0 ** -133, F16: 2.0 ** -24}[t.dtype]
    assert ((got.double() - want).abs() <= bound).all()


SIZES = [
    ([1], [F32]), ([7], [BF]), ([8, 0, 1, 16384, 16385], [F32]), ([100003], [F16]),
    ([3, 70000, 5, 33333, 1, 1, 250000], [BF, F32, F16]), ([1000] * 700, [BF, F32]),
    ([17] * 513, [F16]),
]


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("sizes,dtypes", SIZES)
def test_norm_and_clip(sizes, dtypes, p):
    ts = make(sizes, dtypes, len(sizes))
    want = norm_of(ts, p)
    close(tt.grad_norm(ts, p), want)
    before = [t.clone() for t in ts]
    for max_norm in (float(want) * 0.37, float(want) * 10):
        out = [torch.full_like(t, 7.0) for t in ts]
        close(tt.clip_grad_norm(ts, max_norm, norm_type=p, out=out), want)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
        for o, t in zip(out, ts):
            scaled(o, t, want, max_norm)
    close(tt.clip_grad_norm(ts, float(want) * 10, norm_type=p), want)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))       # in place, nothing to do
    close(tt.clip_grad_norm(ts, float(want) * 0.1, norm_type=p), want)
    for t, b in zip(ts, before):
        scaled(t, b, want, float(want) * 0.1)


@pytest.mark.parametrize("scale,dtype", [(1e30, F32), (1e-30, F32), (1e38, BF), (1e-38, BF),
                                         (3e4, F16), (6e-8, F16), (1e-42, F32)])
def test_squares_outside_fp32(scale, dtype):
    ts = make([4000, 33], [dtype], 1, scale)
    ts = [t.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max) for t in ts]
    for p in (2.0, 1.0, INF):
        want = float(norm_of(ts, p))
        got = float(tt.grad_norm(ts, p))
        assert got == INF if want > torch.finfo(F32).max else \
            abs(got - want) <= 16 * EPS * want + 2.0 ** -149


def test_zeros_and_one_value():
    z = [torch.zeros(5000, device=DEV, dtype=BF), torch.zeros(3, device=DEV)]
    assert float(tt.grad_norm(z)) == 0.0
    z[0][4321] = -3.0
    for p in (1.0, 2.0, INF):
        assert float(tt.grad_norm(z, p)) == 3.0
    assert float(tt.grad_norm([z[0][:0]])) == 0.0
    assert float(tt.clip_grad_norm([z[0][:0]], 1.0)) == 0.0


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_nan_and_infinity(p):
    ts = make([1000, 50], [F32], 2)
    ts[1][17] = INF
    assert float(tt.grad_norm(ts, p)) == INF
    out = [torch.empty_like(t) for t in ts]
    tt.clip_grad_norm(ts, 1.0, norm_type=p, out=out)
    assert not out[0].any() and out[1][17].isnan()                 # g * 0, inf * 0
    ts[0][3] = math.nan
    assert math.isnan(float(tt.grad_norm(ts, p)))
    tt.clip_grad_norm(ts, 1.0, norm_type=p)
    assert ts[0].isnan().all()


def test_off_boundaries_and_strides():
    base = make([4000], [BF], 3)[0]
    views = [base[1:777], base[778:1780], base[1783:1784], base[2000:2600].view(20, 30).t()]
    want = norm_of(views, 2.0)
    copies = [v.clone() for v in views]
    close(tt.grad_norm(views), want)
    gap = base[::2]
    close(tt.grad_norm([gap]), norm_of([gap], 2.0))
    out = make([5000], [BF], 4)[0]
    outs = [out[4:780], out[801:1803], out[1900:1901], out[2001:2601].view(20, 30).t()]
    tt.clip_grad_norm(views, 2.0, out=outs)
    for o, v in zip(outs, views):
        scaled(o, v, want, 2.0)
    tt.clip_grad_norm(views, 2.0)
    for v, c in zip(views, copies):
        scaled(v, c, want, 2.0)
    # what lies between the views is as it was
    again = make([4000], [BF], 3)[0]
    for a, b in ((0, 1), (777, 778), (1780, 1783), (1784, 2000), (2600, 4000)):
        assert torch.equal(base[a:b], again[a:b])


def test_a_norm_of_the_callers():
    ts = make([3000], [F32], 5)
    given = torch.full((1,), 50.0, device=DEV)
    before = ts[0].clone()
    assert float(tt.clip_grad_norm(ts, 5.0, norm=given)) == 50.0
    scaled(ts[0], before, 50.0, 5.0)


def test_same_bits_and_replay():
    ts = make([100000, 3, 50001], [BF, F32], 6)
    a, b = tt.grad_norm(ts), tt.grad_norm(ts)
    assert torch.equal(a, b)
    out = [torch.empty_like(t) for t in ts]
    tt.clip_grad_norm(ts, 1.0, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = tt.clip_grad_norm(ts, 1.0, out=out)
    for t in ts:
        t.mul_(2)
    graph.replay()
    close(norm, norm_of(ts, 2.0))
    for o, t in zip(out, ts):
        scaled(o, t, norm_of(ts, 2.0), 1.0)


def test_autograd_sees_the_write():
    w = torch.ones(4, device=DEV, requires_grad=True)
    x = torch.full((4,), 3.0, device=DEV)
    y = (w * x).sum()
    tt.clip_grad_norm([x], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    t = make([10, 10], [F32])
    for bad in (dict(norm_type=3.0), dict(norm_type=-INF), dict(eps=-1.0), dict(eps=INF),
                dict(out=t[:1]), dict(out=[t[0], t[1].bfloat16()]), dict(out=[t[0], t[1][:5]]),
                dict(out=[t[0], t[0]]), dict(out=[t[1], t[0]])):
        with pytest.raises(ValueError):
            tt.clip_grad_norm(t, 1.0, **bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            tt.clip_grad_norm(t, bad)
    with pytest.raises(ValueError):
        tt.clip_grad_norm([t[0], t[0]], 1.0)               # the same tensor twice
    with pytest.raises(ValueError):
        tt.clip_grad_norm([t[0][:6], t[0][5:]], 1.0)       # overlapping ones
    with pytest.raises(ValueError):
        tt.clip_grad_norm([t[0][::2]], 1.0)
    with pytest.raises(ValueError):
        tt.clip_grad_norm([t[0][:1].expand(10)], 1.0)
    with pytest.raises(ValueError):
        tt.grad_norm([])
    with pytest.raises(TypeError):
        tt.grad_norm([t[0].double()])
    with pytest.raises(TypeError):
        tt.clip_grad_norm(t, 1.0, norm=torch.ones(1, device=DEV, dtype=torch.float64))
    with pytest.raises(RuntimeError):
        tt.grad_norm([t[0], t[1].cpu()])
    assert float(tt.grad_norm([t[0], t[0]])) == pytest.approx(float(t[0].norm()) * 2 ** 0.5, rel=1e-6)


def test_a_norm_among_the_written():
    flat = torch.ones(40, device="cuda")
    with pytest.raises(ValueError):
        tt.clip_grad_norm([flat[:30]], 1.0, norm=flat[29:30])
    with pytest.raises(ValueError):
        tt.clip_grad_norm([flat[:10]], 1.0, norm=flat[20:21], out=[flat[20:30]])
    tt.clip_grad_norm([flat[:30]], 0.5, norm=flat[30:31], eps=0.0)
    assert torch.equal(flat, torch.tensor([0.5] * 30 + [1.0] * 10, device="cuda"))
