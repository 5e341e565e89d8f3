"""``expert_plan`` / ``expert_dispatch`` / ``expert_combine`` against plain
indexing on the CPU: the sort exactly, sums in 64 bits.

Bounds: a combined value is a chain of k fp32 multiply-adds over sum |w y|
(steps = k + 1); a weight's gradient a sum of H products (steps = H); a
dispatched row is a copy, its gradient a chain of k sums.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check, directional

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def sorted_plan(ids, E):
    """slots, entries, offsets of a stable sort, in plain Python"""
    T, k = ids.shape
    flat = ids.reshape(-1).tolist()
    slots, entries, offsets = [-1] * (T * k), [], [0]
    for e in range(E):
        for i, f in enumerate(flat):
            if f == e:
                slots[i] = len(entries)
                entries.append(i)
        offsets.append(len(entries))
    entries += [-1] * (T * k - len(entries))
    return torch.tensor(slots).view(T, k), torch.tensor(entries), torch.tensor(offsets)


def ids_of(T, k, E, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "random":
        return torch.randint(0, E, (T, k), generator=g)
    if kind == "one":
        return torch.full((T, k), E - 1)
    if kind == "none":
        return torch.full((T, k), -1)
    return torch.randint(-2, E + 2, (T, k), generator=g)        # some dropped, on both sides


@pytest.mark.parametrize("kind", ["random", "one", "none", "dropped"])
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (47, 2, 4), (1, 8, 256), (33, 3, 7), (700, 4, 40),
                                   (2047, 2, 5), (5000, 1, 3)])
@pytest.mark.parametrize("itype", [torch.int64, torch.int32])
def test_plan(T, k, E, kind, itype):
    ids = ids_of(T, k, E, kind)
    p = tt.expert_plan(ids.to(itype).to(DEV), E)
    s, n, o = sorted_plan(ids, E)
    assert torch.equal(p.slots.cpu().long(), s)
    assert torch.equal(p.entries.cpu().long(), n)
    assert torch.equal(p.offsets.cpu().long(), o)
    assert torch.equal(p.counts.cpu().long(), o[1:] - o[:-1])


@pytest.mark.parametrize("T,k,E", [(32768, 8, 256), (100003, 3, 1024), (400000, 1, 17)])
def test_large_plans(T, k, E):
    ids = ids_of(T, k, E, "dropped", 3)
    p = tt.expert_plan(ids.to(DEV), E)
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    order = torch.sort(key, stable=True).indices
    kept = int((key < E).sum())
    entries = p.entries.cpu().long()
    assert torch.equal(entries[:kept], order[:kept]) and (entries[kept:] == -1).all()
    assert int(p.offsets[-1]) == kept
    slots = p.slots.cpu().long().reshape(-1)
    assert torch.equal(slots[order[:kept]], torch.arange(kept))
    assert (slots[order[kept:]] == -1).all()
    assert torch.equal(p.counts.cpu().long(), torch.bincount(key, minlength=E + 1)[:E])


@pytest.mark.parametrize("kind", ["random", "dropped", "none"])
@pytest.mark.parametrize("T,k,E,H,dtype,wdtype", [
    (1, 1, 1, 1, F32, F32), (47, 2, 4, 128, F32, F32), (130, 8, 32, 2048, BF, F32),
    (65, 3, 7, 77, F16, F16), (33, 11, 16, 520, BF, BF), (20, 4, 8, 8192, BF, F32),
    (300, 2, 5, 64, F16, F32), (9, 1, 3, 4100, F32, BF), (17, 17, 40, 96, BF, F32),
    (11, 64, 90, 32, F32, BF), (5, 33, 40, 5000, BF, F16),
])
def test_there_and_back(T, k, E, H, dtype, wdtype, kind):
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    ids = ids_of(T, k, E, kind)
    slots, entries, offsets = sorted_plan(ids, E)
    kept = int(offsets[-1])
    plan = tt.expert_plan(ids.to(DEV), E)
    x, ys = r(T, H).to(dtype).requires_grad_(True), r(T * k, H).to(dtype).requires_grad_(True)
    w = torch.rand(T, k, generator=g, device=DEV).to(wdtype).requires_grad_(True)
    dxs, dy = r(T * k, H).to(dtype), r(T, H).to(dtype)
    xs = tt.expert_dispatch(x, plan)
    y = tt.expert_combine(ys, w, plan)
    dx, dw, dys = torch.autograd.grad([xs, y], [x, w, ys], [dxs, dy])
    for a, b in ((xs, ys), (dys, ys), (dx, x), (dw, w), (y, x)):
        assert a.dtype == b.dtype and a.shape == b.shape
    # 64 bits, on the CPU
    c = lambda t: t.detach().double().cpu()
    at, there = slots.clamp(min=0), (slots >= 0)
    want = torch.zeros(T * k, H, dtype=torch.float64)
    want[:kept] = c(x)[entries[:kept] // k]
    assert torch.equal(c(xs), want)
    wk = c(w) * there
    terms = wk[..., None] * c(ys)[at]
    check("y", y.detach(), terms.sum(1), terms.abs().sum(1), k + 1)
    terms = c(dxs)[at] * there[..., None]
    check("dx", dx, terms.sum(1), terms.abs().sum(1), k)
    terms = c(ys)[at] * c(dy)[:, None] * there[..., None]
    check("dw", dw, terms.sum(-1), terms.abs().sum(-1), H)
    want = torch.zeros(T * k, H, dtype=torch.float64)
    e = entries[:kept]
    want[:kept] = c(w).reshape(-1)[e][:, None] * c(dy)[e // k]
    check("dys", dys, want, want.abs(), 1)


def test_rows_off_their_alignment():
    ids = ids_of(50, 2, 6, "random").to(DEV)
    plan = tt.expert_plan(ids, 6)
    buf = torch.randn(1 + 50 * 64, device=DEV).to(BF)
    x = buf[1:].view(50, 64)
    assert x.data_ptr() % 16
    assert torch.equal(tt.expert_dispatch(x, plan), tt.expert_dispatch(x.clone(), plan))
    wide = torch.randn(50, 128, device=DEV).to(BF)
    assert torch.equal(tt.expert_dispatch(wide[:, :64], plan),
                       tt.expert_dispatch(wide[:, :64].contiguous(), plan))


def test_nothing_of_a_dropped_choice_is_read():
    ids = torch.tensor([[0, -1], [1, 5]], device=DEV)
    plan = tt.expert_plan(ids, 2)
    ys = torch.full((4, 8), float("nan"), device=DEV)
    ys[:2] = 1.0
    w = torch.tensor([[0.5, float("nan")], [2.0, float("inf")]], device=DEV, requires_grad=True)
    y = tt.expert_combine(ys, w, plan)
    assert torch.equal(y, torch.tensor([[0.5], [2.0]], device=DEV).expand(2, 8))
    dw, = torch.autograd.grad(y.sum(), [w])
    assert torch.equal(dw, torch.tensor([[8.0, 0.0], [8.0, 0.0]], device=DEV))


def test_gradients_by_differences():
    # linear in each input: differences are exact up to rounding
    ids = ids_of(12, 3, 5, "dropped").to(DEV)
    plan = tt.expert_plan(ids, 5)
    x = torch.randn(12, 40, device=DEV, requires_grad=True)
    wx = torch.randn(36, 40, device=DEV)
    directional(lambda t: [tt.expert_dispatch(t, plan)], [x], [wx],
                torch.autograd.grad(tt.expert_dispatch(x, plan), [x], [wx]), 0.5, 1e-3)
    ys = torch.randn(36, 40, device=DEV, requires_grad=True)
    w = torch.rand(12, 3, device=DEV, requires_grad=True)
    wy = torch.randn(12, 40, device=DEV)
    # bilinear in (ys, w): the central difference has no second-order error
    directional(lambda a, b: [tt.expert_combine(a, b, plan)], [ys, w], [wy],
                torch.autograd.grad(tt.expert_combine(ys, w, plan), [ys, w], [wy]), 0.5, 1e-3)


def test_same_result_twice_and_on_another_stream():
    ids = ids_of(4000, 4, 16, "random").to(DEV)
    ys, w = torch.randn(16000, 256, device=DEV).to(BF), torch.rand(4000, 4, device=DEV)

    def go():
        plan = tt.expert_plan(ids, 16)
        return plan.entries, tt.expert_combine(ys, w, plan)
    a = go()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = go()
    s.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("T,k", [(0, 4), (5, 0), (0, 0)])
def test_nothing_to_sort(T, k):
    plan = tt.expert_plan(torch.zeros(T, k, dtype=torch.int64, device=DEV), 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0] and plan.slots.shape == (T, k)
    x = torch.randn(T, 16, device=DEV, requires_grad=True)
    xs = tt.expert_dispatch(x, plan)
    assert xs.shape == (0, 16)
    w = torch.rand(T, k, device=DEV, requires_grad=True)
    y = tt.expert_combine(xs, w, plan)
    assert torch.equal(y, torch.zeros(T, 16, device=DEV))
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert not dx.any() and dw.shape == (T, k)


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError):
        tt.expert_plan(ids.cpu(), 4)
    with pytest.raises(TypeError):
        tt.expert_plan(ids.float(), 4)
    for a in ((ids[0], 4), (ids, 0), (ids, 1025), (ids[:, :1].expand(4, 65), 4)):
        with pytest.raises(ValueError):
            tt.expert_plan(*a)
    plan = tt.expert_plan(ids, 4)
    x, ys, w = (torch.randn(*s, device=DEV) for s in ((4, 8), (8, 8), (4, 2)))
    with pytest.raises(RuntimeError):
        tt.expert_dispatch(x.cpu(), plan)
    with pytest.raises(RuntimeError):
        tt.expert_combine(ys, w.cpu(), plan)
    with pytest.raises(TypeError):
        tt.expert_dispatch(x.double(), plan)
    with pytest.raises(TypeError):
        tt.expert_combine(ys, w.double(), plan)
    for f in (lambda: tt.expert_dispatch(x[:3], plan), lambda: tt.expert_dispatch(x[0], plan),
              lambda: tt.expert_dispatch(x[:, :0], plan), lambda: tt.expert_combine(x, w, plan),
              lambda: tt.expert_combine(ys, w[:, :1], plan)):
        with pytest.raises(ValueError):
            f()


def test_differentiating_twice_is_refused():
    plan = tt.expert_plan(torch.zeros(4, 2, dtype=torch.int64, device=DEV), 2)
    ys = torch.randn(8, 16, device=DEV, requires_grad=True)
    w = torch.rand(4, 2, device=DEV)
    g, = torch.autograd.grad(tt.expert_combine(ys, w, plan).sum(), [ys], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [ys])


def test_leaf_gradients_add_up():
    plan = tt.expert_plan(torch.tensor([[0], [1], [0]], device=DEV), 2)
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    for _ in range(2):
        tt.expert_dispatch(x, plan).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))


@pytest.mark.parametrize("H", [2048, 2047])
def test_offsets_over_32_bits(H):
    # 2^31 elements and more of sorted rows; the last expert's rows lie behind them
    T, k, E = (1 << 31) // (4 * H) + 40, 4, 4
    ids = torch.arange(4, device=DEV).expand(T, 4).contiguous()
    plan = tt.expert_plan(ids, E)
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.zeros(T, H, dtype=BF, device=DEV)
    rows = [0, T // 2, T - 1]
    x[rows] = torch.randn(3, H, generator=g, device=DEV).to(BF)
    x.requires_grad_(True)
    w = torch.rand(T, k, generator=g, device=DEV, requires_grad=True)
    xs = tt.expert_dispatch(x, plan)
    for e in range(E):
        assert torch.equal(xs[[e * T + r for r in rows]], x[rows])
    y = tt.expert_combine(xs, w, plan)
    wr, xr = w[rows].detach().double(), x[rows].detach().double()
    check("y", y[rows].detach(), wr.sum(1, keepdim=True) * xr, wr.sum(1, keepdim=True) * xr.abs(), 5)
    dy = torch.zeros_like(y)
    dy[rows] = torch.randn(3, H, generator=g, device=DEV).to(BF)
    dw, = torch.autograd.grad(y, [w], [dy])
    dot = dy[rows].double() * xr
    check("dw", dw[rows], dot.sum(1, keepdim=True).expand(3, 4),
          dot.abs().sum(1, keepdim=True).expand(3, 4), H)
