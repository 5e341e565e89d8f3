"""The LM head's loss without logits, and its gradients, against the formulas in 64
bits.

Bounds.  A logit is off by at most 2 H 2^-24 of the sum of its terms' magnitudes (the
tensor cores cut off where fp32 rounds).  Losses and lse take that of the largest
logit's error, and the sum of V exponentials of tiles joined two by two.  dz is
rounded to the inputs' type once: u(T) of each through the product's magnitudes.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import EPS, TINY, UNIT, directional

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def make(T, H, V, M, dtype, seed=0, size=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, w = r(T, H).to(dtype), (r(V, H) * size * H ** -0.5).to(dtype)
    labels = torch.randint(0, V, (T, M), generator=g, device=DEV)
    labels[:, 1:][torch.rand(T, M - 1, generator=g, device=DEV) < 0.5] = -100
    labels[2::5] = V + 3
    return x, w, labels, torch.rand(T, M, generator=g, device=DEV) / T, r(T) * 0.1 / T


def compare(x, w, labels, gl, ge, scale=1.0):
    leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
    r = tt.linear_cross_entropy(*leaves, labels, scale=scale)
    assert r.losses.shape == labels.shape and r.lse.shape == x.shape[:1]
    outs, gs = [r.losses, r.lse], [gl.view_as(r.losses), ge]
    dx, dw = torch.autograd.grad(outs, leaves, gs)
    tt.check_device_status()
    x, w = x.detach().double(), w.detach().double()
    T, H = x.shape
    V, lab, gl, ge = w.shape[0], labels.view(T, -1), gl.view(T, -1).double(), ge.double()
    z = scale * (x @ w.t())
    ez = 2 * H * EPS * abs(scale) * (x.abs() @ w.abs().t()) + 2 * EPS * z.abs()
    lse = torch.logsumexp(z, 1)
    ok = (lab >= 0) & (lab < V)
    at = lab.clamp(0, V - 1)
    loss = torch.where(ok, lse[:, None] - z.gather(1, at), 0.0)
    # the sum's roundings: 32 a chunk, the chunks, the joined tiles, exp's own
    top = ez.amax(1) + 128 * EPS + 4 * EPS * z.abs().amax(1)
    for name, got, want, e in (("lse", r.lse, lse, top),
                               ("losses", r.losses.view(T, -1), loss, top[:, None] + ez.gather(1, at))):
        over = (got.detach().double() - want).abs() - e - 4 * EPS * want.abs()
        assert over.max() <= 0, f"{name}: over its bound by {float(over.max()):.3e}"
    assert not r.losses.view(T, -1)[~ok].any()
    p = torch.exp(z - lse[:, None])
    g = torch.where(ok, gl, 0.0)
    dz = p * (g.sum(1) + ge)[:, None]
    dz.scatter_add_(1, at, -g)
    dz *= scale
    ep = p * (ez + top[:, None] + 8 * EPS)
    most = (g.abs().sum(1) + ge.abs())[:, None] * abs(scale)
    t = dx.dtype
    # (fp16: dz is held as multiples of 2^-24 of a power of two over the largest weight)
    edz = most * (ep + 8 * EPS * p) + (UNIT[t] if t != F32 else 2 * EPS) * dz.abs() + \
        EPS * torch.zeros_like(dz).scatter_add_(1, at, g.abs() * abs(scale))
    if t == F16:
        edz = edz + float(most.max()) * 2.0 ** -37
    for name, got, want, e in (
            ("dx", dx, dz @ w, edz @ w.abs() + 2 * (V + 64) * EPS * (dz.abs() @ w.abs())),
            ("dw", dw, dz.t() @ x, edz.t() @ x.abs() + 2 * T * EPS * (dz.abs().t() @ x.abs()))):
        over = (got.double() - want).abs() - UNIT[t] * want.abs() - e - TINY[t]
        assert over.max() <= 0, f"{name}: over its bound by {float(over.max()):.3e}"
    return r, dx, dw


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("T,H,V,M", [
    (1, 1, 1, 1), (1, 64, 300, 1), (47, 256, 3000, 2), (128, 64, 256, 1), (129, 72, 257, 3),
    (300, 200, 1001, 4), (257, 1001, 515, 1), (3, 33, 20001, 1), (1000, 136, 2050, 2)])
def test_losses_and_gradients(T, H, V, M, dtype):
    compare(*make(T, H, V, M, dtype, T + V))


@pytest.mark.parametrize("dtype,T,V", [(BF, 33000, 9001), (F16, 40000, 4500), (F32, 20000, 8500)])
def test_several_pieces_of_the_vocabulary(dtype, T, V):
    compare(*make(T, 40, V, 1, dtype, 1))


@pytest.mark.parametrize("T,H,V", [(1, 2560, 30000), (20, 512, 151936), (5, 5120, 4000)])
def test_long_sides(T, H, V):
    compare(*make(T, H, V, 1, BF, 2))


@pytest.mark.parametrize("scale", [0.25, -1.5, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scale(scale, dtype):
    compare(*make(60, 64, 700, 2, dtype, 3), scale=scale)


def test_labels():
    x, w, _, _, ge = make(64, 48, 600, 1, BF, 4)
    g = torch.rand(64, 9, device=DEV)
    same = torch.full((64, 9), 77, device=DEV)                    # one label many times
    compare(x, w, same, g, ge)
    compare(x, w, torch.randint(0, 600, (64, 9), device=DEV), g, ge)
    compare(x, w, torch.full((64, 9), -100, device=DEV), g, ge)   # none
    compare(x, w, torch.randint(-300, 900, (64,), device=DEV), g[:, 0].contiguous(), ge)
    r = tt.linear_cross_entropy(x, w, torch.empty(64, 0, dtype=torch.int64, device=DEV))
    assert r.losses.shape == (64, 0)
    a = tt.linear_cross_entropy(x, w, same.int())
    assert torch.equal(a.losses, tt.linear_cross_entropy(x, w, same).losses)
    # offsets of a padded array of many successors
    many = torch.full((64, 300), -1, device=DEV)
    many[:, 250] = torch.arange(64, device=DEV)
    compare(x, w, many, torch.rand(64, 300, device=DEV), ge)


def test_one_gradient_only():
    x, w, labels, gl, ge = make(90, 64, 500, 1, BF, 5)
    _, dx, dw = compare(x, w, labels[:, 0].contiguous(), gl[:, 0].contiguous(), ge * 0)
    lab = labels[:, 0]
    for i, want in ((0, dx), (1, dw)):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w))]
        got, = torch.autograd.grad(tt.linear_cross_entropy(*leaves, lab).losses, leaves[i],
                                   gl[:, 0])
        assert torch.equal(got, want)
    # through lse alone
    xs = x.float().clone().requires_grad_(True)
    r = tt.linear_cross_entropy(xs, w.float(), lab)
    got, = torch.autograd.grad(r.lse.sum(), xs)
    p = torch.softmax(x.double() @ w.double().t(), 1)
    assert float((got.double() - p @ w.double()).abs().max()) < 64 * 500 * EPS


def test_weights_far_below_one_in_fp16():
    x, w, labels, gl, ge = make(100, 64, 2000, 1, F16, 6)
    compare(x, w, labels, gl * 1e-2, ge * 1e-2)


def test_strides():
    x, w, labels, gl, ge = make(70, 64, 400, 1, BF, 7)
    wide = torch.randn(400, 150, device=DEV).to(BF)
    compare(wide[:70, 16:80], w, labels, gl, ge)
    compare(wide[:70, 5:69], wide[:, 1:65], labels, gl, ge)
    compare(torch.randn(64, 70, device=DEV).to(BF).t(), w, labels, gl, ge)
    compare(x.float(), wide.float()[:, 3:67], labels, gl, ge)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_rows(dtype):
    x, w, labels, _, _ = make(1, 16, 24, 1, dtype)
    leaves = [x[:0].requires_grad_(True), w.requires_grad_(True)]
    r = tt.linear_cross_entropy(*leaves, labels[:0])
    assert r.losses.shape == (0, 1)
    dx, dw = torch.autograd.grad(r.losses.sum(), leaves)
    assert dx.shape == (0, 16) and not dw.any()


def test_large_logits():
    x, w, labels, gl, ge = make(50, 64, 300, 1, F32, 8, size=300.0)
    compare(x, w, labels, gl, ge)
    r = tt.linear_cross_entropy(x.to(BF), w.to(BF), labels)
    assert r.losses.isfinite().all() and (r.losses >= 0).all()


def test_nan_stays_in_its_row():
    x, w, labels, _, _ = make(140, 64, 300, 1, BF, 9)
    labels = labels.clamp(0, 299)
    clean = tt.linear_cross_entropy(x, w, labels)
    x[70, 3] = float("nan")
    r = tt.linear_cross_entropy(x, w, labels)
    assert r.lse[70].isnan() and r.losses[70].isnan().all()
    rest = torch.arange(140, device=DEV) != 70
    assert torch.equal(r.lse[rest], clean.lse[rest])


def test_differences():
    x, w, labels, gl, ge = make(12, 17, 90, 2, F32, 10)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    f = lambda *a: list(tt.linear_cross_entropy(*a, labels))
    outs = [gl * 12, ge * 12]
    grads = torch.autograd.grad(f(*leaves), leaves, outs)
    # central differences of step s: s^2 / 6 of the third derivative and 2^-24 of the
    # values over s, with s = 2^-6 both under 2e-3 of the gradients' norm
    directional(f, leaves, outs, grads, 2.0 ** -6, 2e-3)


def test_same_bits_another_stream_and_replay():
    x, w, labels, gl, ge = make(333, 128, 1500, 2, BF, 11)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]

    def step():
        r = tt.linear_cross_entropy(*leaves, labels)
        return [r.losses.detach(), *torch.autograd.grad([r.losses, r.lse], leaves, [gl, ge])]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(x.flip(0))
    labels.copy_(labels.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), got))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_backward_twice(dtype):
    x, w, labels, gl, ge = make(70, 64, 500, 2, dtype, 12)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    r = tt.linear_cross_entropy(*leaves, labels)
    one = torch.autograd.grad([r.losses, r.lse], leaves, [gl, ge], retain_graph=True)
    two = torch.autograd.grad([r.losses, r.lse], leaves, [gl, ge])
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_refusals():
    x, w, labels, _, _ = make(4, 16, 24, 1, BF)
    for bad in ((x[0], w, labels), (x, w[:, :8], labels), (x, w, labels[:3]),
                (x, w, labels.view(2, 2, 1))):
        with pytest.raises(ValueError):
            tt.linear_cross_entropy(*bad)
    with pytest.raises(ValueError):
        tt.linear_cross_entropy(x, w, labels, scale=float("nan"))
    with pytest.raises(TypeError):
        tt.linear_cross_entropy(x, w.half(), labels)
    with pytest.raises(TypeError):
        tt.linear_cross_entropy(x, w, labels.float())
    with pytest.raises(RuntimeError):
        tt.linear_cross_entropy(x, w, labels.cpu())


@pytest.mark.parametrize("dtype,T,H,V,M", [(BF, 15, 72, 1001, 3), (F16, 9, 130, 777, 2),
                                           (BF, 300, 1024, 2050, 2), (F16, 260, 1032, 515, 9),
                                           (BF, 1, 2560, 40001, 300)])
def test_16_bit_logits_that_are_left_for_the_backward(dtype, T, H, V, M):
    from tree_training_b200 import _lib
    assert _lib.lib().tt_linear_ce_kept_ld({BF: 1, F16: 2}[dtype], T, H, V)
    compare(*make(T, H, V, M, dtype, T))
    x, w, _, gl, ge = make(T, H, V, M, dtype, T)
    compare(x, w, torch.full((T, M), V - 1, device=DEV), gl, ge)        # one label for all


def test_widths_that_32_bits_do_not_count():
    one = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16)
    wide = one.expand(1, (1 << 31) - 257)
    with pytest.raises(ValueError):
        tt.linear_cross_entropy(wide, wide, torch.zeros(1, device="cuda", dtype=torch.int64))
    with pytest.raises(ValueError):
        tt.linear_cross_entropy(one, one.expand((1 << 31) - 256, 1),
                                torch.zeros(1, device="cuda", dtype=torch.int64))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 7, 8, 13, 16, 17])
@pytest.mark.parametrize("H,V", [(1001, 735), (2048, 333), (96, 20001)])
def test_few_rows_of_fp32(T, H, V):
    compare(*make(T, H, V, 2, torch.float32, seed=T))
