"""``residual_norm`` against its definition in 64 bits (gradients by
differentiation in 64 bits): every gate, norms on one side and both, fp32 and
16-bit streams, widths that are odd, tiny and over one block's registers.

Bounds.  A row's mean square is a sum of D fp32 terms whose longest chain is 16
(a thread's) + 5 (a warp's) + 32 (the warps'); with the reciprocal root (2 ulp)
and the products around it under 96 roundings: steps = 96 for y and r over
|residual| + |scale g h|, and 3 * 96 for the gradients, which go through both
norms.  A weight's gradient also adds one term a row: steps + rows.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check, directional

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def data(T, D, dtype, res, post, gate, wdtype=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    wdtype = wdtype or dtype
    v = {"x": (r(T, D) * 0.8).to(dtype)}
    if res is not None:
        v["residual"] = (r(T, D) * 2).to(res)
    v["weight"] = (1 + 0.2 * r(D)).to(wdtype)
    if post:
        v["post_weight"] = (1 + 0.2 * r(D)).to(wdtype)
    shape = {"none": None, "channel": (D,), "row": (T, 1), "full": (T, D)}[gate]
    if shape:
        v["gate"] = torch.sigmoid(r(*shape)).to(dtype)
    dy = r(T, D).to(dtype)
    dr = r(T, D).to(res or dtype)
    return v, dy, dr


def op(v, **kw):
    return tt.residual_norm(v["x"], v.get("residual"), v["weight"],
                            post_weight=v.get("post_weight"), gate=v.get("gate"), **kw)


def reference(v, scale, eps, offset):
    """(y, r, magnitude of r, factor from r to y) in 64 bits"""
    rms = lambda t: torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)
    h = v["x"]
    if "post_weight" in v:
        h = h * rms(h) * (offset + v["post_weight"])
    b = scale * (h * v["gate"] if "gate" in v else h)
    res = v.get("residual")
    r = b if res is None else res + b
    f = rms(r) * (offset + v["weight"])
    return r * f, r, b.abs() + (0 if res is None else res.abs()), f


def run(T, D, dtype, res, post, gate, scale=1.0, offset=0.0, eps=1e-6, wdtype=None, edit=None):
    v, dy, dr = data(T, D, dtype, res, post, gate, wdtype)
    if edit:
        edit(v)
    for t in v.values():
        t.requires_grad_(True)
    y, r = op(v, scale=scale, eps=eps, weight_offset=offset)
    assert y.dtype == dtype and r.dtype == (res or dtype)
    got = torch.autograd.grad([y, r], list(v.values()), [dy, dr])
    d = {n: t.detach().double().requires_grad_(True) for n, t in v.items()}
    yw, rw, mag, f = reference(d, scale, eps, offset)
    want = torch.autograd.grad([yw, rw], list(d.values()), [dy.double(), dr.double()])
    check("r", r.detach(), rw.detach(), mag.detach(), 96)
    check("y", y.detach(), yw.detach(), (mag * f.abs()).detach(), 96)
    with torch.no_grad():
        x, w = d["x"], offset + d["weight"]
        i2 = torch.rsqrt(rw.square().mean(-1, keepdim=True) + eps)
        gy, n = dy.double() * w, rw * i2
        an = mag * i2                                # |n|, cancellation in r counted
        ddr = dr.double().abs() + i2 * (gy.abs() + an * (gy.abs() * an).mean(-1, keepdim=True))
        i1 = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) if post else 1.0
        w1 = (offset + d["post_weight"]).abs() if post else 1.0
        gt = d["gate"].abs() if "gate" in d else 1.0
        h = x.abs() * i1 * w1
        dh = abs(scale) * gt * ddr
        dx = i1 * dh * w1
        if post:
            n1 = x.abs() * i1
            dx = dx + i1 * n1 * (dh * w1 * n1).mean(-1, keepdim=True)
        mags = {"x": dx, "residual": ddr, "weight": (dy.double().abs() * an).sum(0)}
        if post:
            mags["post_weight"] = (dh * x.abs() * i1).sum(0)
        if "gate" in d:
            dg = abs(scale) * h * ddr
            mags["gate"] = {"channel": dg.sum(0), "row": dg.sum(1, keepdim=True), "full": dg}[gate]
    for name, a, b in zip(v, got, want):
        assert a.dtype == v[name].dtype and a.shape == v[name].shape
        rows = T if name in ("weight", "post_weight") or gate == "channel" else 0
        check("d" + name, a, b, mags[name], 288 + rows)


@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("T,D,dtype,res", [
    (47, 256, F32, F32), (130, 2560, BF, BF), (33, 320, F16, F16), (19, 520, BF, F32),
    (21, 129, BF, BF), (300, 4608, BF, BF), (31, 1026, F16, F16), (5, 1001, F32, F32), (300, 64, F16, F32), (7, 24, BF, BF),
])
def test_every_form(T, D, dtype, res, post, gate):
    run(T, D, dtype, res, post, gate, scale=0.5, offset=1.0 if post else 0.0)


@pytest.mark.parametrize("T,D,dtype", [
    (2500, 640, BF), (700, 5120, F16), (40, 6152, F32), (1500, 1032, BF), (2000, 2560, F32), (1300, 4096, BF), (1, 1, F32), (3, 2, BF), (1, 4096, BF), (2, 4097, F16), (5, 4104, F32), (6, 8192, BF),
    (3, 8200, BF), (2, 16384, F32), (2, 16383, BF), (1500, 40, BF), (5000, 128, BF),
])
@pytest.mark.parametrize("full", [False, True])
def test_widths(T, D, dtype, full):
    run(T, D, dtype, dtype, full, "full" if full else "none")


def test_no_residual_and_weights_in_32_bits():
    run(50, 384, BF, None, False, "none")
    run(50, 384, BF, None, True, "row", scale=2.0)
    run(50, 384, BF, F32, True, "full", wdtype=F32)
    run(50, 384, F16, F16, False, "none", wdtype=F32)


def test_rows_of_zeros_large_eps_and_large_values():
    def edit(v):
        v["x"][3] = 0
        v["residual"][3] = 0
        v["x"][4] *= 1000
        v["residual"][5] *= 1000
    run(12, 640, F32, F32, True, "none", edit=edit)
    run(12, 640, BF, BF, False, "channel", eps=0.5, edit=edit)


def test_residual_that_cancels_the_block():
    # r nearly zero: its mean square must not come out of differences of sums
    def edit(v):
        v["residual"].copy_(-0.5 * v["x"] + 1e-3 * v["residual"])
    run(16, 512, F32, F32, False, "none", scale=0.5, edit=edit)


def test_nan_and_infinity_stay_in_their_row():
    v, _, _ = data(9, 256, BF, BF, True, "full")
    y0, r0 = op(v)
    v["x"][2, 7] = float("nan")
    v["residual"][5, 3] = float("inf")
    y, r = op(v)
    keep = [0, 1, 3, 4, 6, 7, 8]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(r[keep], r0[keep])
    assert y[2].isnan().all() and r[5, 3] == float("inf") and y[5, 3].isnan()


def test_strides_and_leading_dims():
    v, dy, dr = data(24, 256, BF, BF, True, "full")
    want = op(v)
    pad = {n: (torch.cat([t, t], 1)[:, :256] if t.dim() == 2 else t) for n, t in v.items()}
    assert all(torch.equal(a, b) for a, b in zip(op(pad), want))
    odd = {n: (torch.cat([t[:, :1], t], 1)[:, 1:] if t.dim() == 2 else t) for n, t in v.items()}
    for a, b in zip(op(odd), want):        # rows off by one element: the unaligned form
        check("unaligned", a, b.double(), b.double().abs(), 2.0 ** 17)
    cube = {n: (t.view(2, 12, 256) if t.dim() == 2 else t) for n, t in v.items()}
    for a, b in zip(op(cube), want):
        assert a.shape == (2, 12, 256) and torch.equal(a.view(24, 256), b)
    turned = {n: (t.t().contiguous().t() if t.dim() == 2 else t) for n, t in v.items()}
    assert all(torch.equal(a, b) for a, b in zip(op(turned), want))


def test_gradient_of_either_output_and_expanded_gradients():
    v, dy, dr = data(30, 256, F32, F32, False, "none")
    for t in v.values():
        t.requires_grad_(True)
    both = torch.autograd.grad(op(v), list(v.values()), [dy, dr])
    only_y = torch.autograd.grad(op(v)[0], list(v.values()), [dy])
    only_r = torch.autograd.grad(op(v)[1], [v["x"], v["residual"]], [dr])
    for name, a, b, c in zip(("x", "residual"), both, only_y, only_r):
        check(name, (b + c), a.double(), b.double().abs() + c.double().abs(), 300)
    assert torch.equal(both[2], only_y[2])
    s, = torch.autograd.grad(op(v)[1].sum(), [v["residual"]])      # an expanded 1
    assert torch.equal(s, torch.ones_like(s))
    w, = torch.autograd.grad(op(v)[0], [v["weight"]], [dy])
    assert torch.equal(w, both[2])


def test_shared_input():
    # x and residual are one tensor: both gradients add up
    v, dy, dr = data(10, 128, F32, F32, False, "none")
    x = v["x"].requires_grad_(True)
    g, = torch.autograd.grad(tt.residual_norm(x, x, v["weight"]), [x], [dy, dr])
    d = x.detach().double().requires_grad_(True)
    yw, rw, _, _ = reference({"x": d, "residual": d, "weight": v["weight"].double()}, 1.0, 1e-6, 0.0)
    w, = torch.autograd.grad([yw, rw], [d], [dy.double(), dr.double()])
    check("dx", g, w, w.abs() + 8, 288)


def test_gradients_by_differences():
    # the central difference is off by h^2 / 6 of the third derivative (1e-4 at
    # h = 1e-2 for values around 1) and by 2^-24 sqrt(n) / h: under 1e-3 of |grad|
    v, dy, dr = data(20, 96, F32, F32, True, "full")
    names = list(v)
    for t in v.values():
        t.requires_grad_(True)
    grads = torch.autograd.grad(op(v, scale=0.7), list(v.values()), [dy, dr])
    f = lambda *ts: op(dict(zip(names, ts)), scale=0.7)
    directional(f, list(v.values()), [dy, dr], grads, 1e-2, 1e-2)


def test_same_result_twice_and_on_another_stream():
    v, dy, dr = data(3000, 256, BF, BF, True, "channel")
    for t in v.values():
        t.requires_grad_(True)
    first = torch.autograd.grad(op(v), list(v.values()), [dy, dr])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = torch.autograd.grad(op(v), list(v.values()), [dy, dr])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_no_rows():
    v, dy, dr = data(0, 64, BF, BF, True, "channel")
    for t in v.values():
        t.requires_grad_(True)
    y, r = op(v)
    assert y.shape == r.shape == (0, 64)
    gs = torch.autograd.grad([y, r], list(v.values()), [dy, dr])
    assert all(not g.any() for g in gs) and gs[2].shape == (64,)


def test_refusals():
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    ok = tt.residual_norm
    with pytest.raises(RuntimeError):
        ok(x.cpu(), None, w)
    with pytest.raises(RuntimeError):
        ok(x, x.cpu(), w)
    with pytest.raises(TypeError):
        ok(x.double(), None, w.double())
    with pytest.raises(TypeError):
        ok(x, x.bfloat16(), w)
    with pytest.raises(TypeError):
        ok(x, x, w.bfloat16())
    with pytest.raises(TypeError):
        ok(x.bfloat16(), None, w, post_weight=w.bfloat16())
    with pytest.raises(TypeError):
        ok(x, x, w, gate=w.bfloat16())
    for kw in (dict(residual=x[:3]), dict(weight=w[:4]), dict(post_weight=w[None]),
               dict(gate=w[:4]), dict(gate=x[:2]), dict(gate=x[:, :2])):
        with pytest.raises(ValueError):
            ok(x, kw.pop("residual", x), kw.pop("weight", w), **kw)
    big = torch.zeros(1, 16385, device=DEV)
    with pytest.raises(ValueError):
        ok(big, None, big[0])


def test_differentiating_twice_is_refused():
    v, dy, dr = data(6, 64, F32, F32, False, "none")
    x = v["x"].requires_grad_(True)
    y, r = op(v)
    gs = torch.autograd.grad([y, r], [x], [dy, dr], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gs[0].sum(), [x])


@pytest.mark.parametrize("D", [4096, 4098])
def test_offsets_over_32_bits(D):
    T = (1 << 31) // D + 70
    rows = [0, 1, T // 2, T - 2, T - 1]
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.ones(T, D, dtype=BF, device=DEV)
    r = torch.zeros(T, D, dtype=BF, device=DEV)
    x[rows] = torch.randn(5, D, generator=g, device=DEV).to(BF)
    r[rows] = torch.randn(5, D, generator=g, device=DEV).to(BF)
    w = torch.ones(D, dtype=BF, device=DEV)
    x.requires_grad_(True)
    y, s = tt.residual_norm(x, r, w, scale=0.5)
    d = {"x": x[rows].detach().double().requires_grad_(True), "residual": r[rows].double(),
         "weight": w.double()}
    yw, rw, mag, f = reference(d, 0.5, 1e-6, 0.0)
    check("r", s[rows].detach(), rw.detach(), mag.detach(), 96)
    check("y", y[rows].detach(), yw.detach(), (mag * f.abs()).detach(), 96)
    dy = torch.zeros_like(y)
    dy[rows] = torch.randn(5, D, generator=g, device=DEV).to(BF)
    dx, = torch.autograd.grad(y, [x], [dy])
    want, = torch.autograd.grad(yw, [d["x"]], [dy[rows].double()])
    i2 = torch.rsqrt(rw.square().mean(-1, keepdim=True) + 1e-6)
    an, gy = mag * i2, dy[rows].double().abs()
    size = 0.5 * i2 * (gy + an * (gy * an).mean(-1, keepdim=True))
    check("dx", dx[rows], want, size.detach(), 288)


@pytest.mark.parametrize("post,gate", [(True, "none"), (True, "row"), (True, "full"),
                                       (True, "channel"), (False, "channel"), (False, "full")])
@pytest.mark.parametrize("D,dtype,res", [
    (1032, BF, BF), (1536, F16, F16), (2576, BF, F32), (4104, BF, BF), (5120, BF, F32),
    (8192, BF, BF), (4104, F32, F32), (5120, F32, F32),
])
def test_many_rows_a_block(D, dtype, res, post, gate):
    # the weights' sums over rows that pass round the stages several times
    run(3001, D, dtype, res, post, gate, scale=0.5)
