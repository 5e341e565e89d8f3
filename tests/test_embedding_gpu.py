"""Embedding rows and the table's gradient against the formulas in 64 bits."""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def make(n, V, H, dtype, seed=0, same=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ids = torch.randint(0, V, (n,), generator=g, device=DEV)
    if same:                                  # one word makes up much of the text
        ids[torch.rand(n, generator=g, device=DEV) < same] = V // 2
    w = torch.randn(V, H, generator=g, device=DEV).to(dtype)
    dy = torch.randn(n, H, generator=g, device=DEV).to(dtype)
    return ids, w, dy


def compare(ids, w, dy, scale=1.0, padding=None, cast=lambda i: i):
    w = w.detach().requires_grad_(True)
    y = tt.embedding(cast(ids), w, scale=scale, padding_idx=padding)
    check("y", y, w.detach().double()[ids] * scale, w.detach().double()[ids].abs() * abs(scale), 2)
    y.backward(dy)
    V, H = w.shape
    flat, d = ids.reshape(-1), dy.reshape(-1, H).double() * scale
    keep = torch.ones_like(flat, dtype=torch.bool) if padding is None else flat != padding % V
    want = torch.zeros(V, H, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], d[keep])
    mag = torch.zeros_like(want).index_add_(0, flat[keep], d[keep].abs())
    # each of a word's n rows goes through at most n additions and the scaling
    most = int(torch.bincount(flat, minlength=V).max()) + 2 if flat.numel() else 2
    check("dw", w.grad, want, mag, most)
    return y, w.grad


@pytest.mark.parametrize("n,V,H,dtype", [
    (1, 1, 1, F32), (47, 32000, 256, F32), (1, 300, 2560, BF), (129, 7, 130, F16),
    (1000, 1023, 1001, BF), (1000, 1025, 64, F16), (4099, 1 << 20, 8, BF),
    (3001, (1 << 20) + 3, 8, F32), (5000, 70000, 72, BF), (33, 50, 8200, F16),
])
def test_rows_and_gradient(n, V, H, dtype):
    compare(*make(n, V, H, dtype, n))


@pytest.mark.parametrize("same", [0.5, 1.0])
@pytest.mark.parametrize("n,H,dtype", [(5000, 72, BF), (2500, 1001, F32), (9000, 640, F16)])
def test_a_word_that_makes_up_the_text(n, H, dtype, same):
    compare(*make(n, 3000, H, dtype, 1, same))


@pytest.mark.parametrize("scale,padding", [(31.6, None), (-0.5, 3), (0.0, 0), (1.0, -1)])
def test_scale_and_padding(scale, padding):
    ids, w, dy = make(700, 40, 96, BF, 2)
    _, dw = compare(ids, w, dy, scale, padding)
    if padding is not None:
        assert not dw[padding].any()


def test_shapes_types_and_strides():
    ids, w, dy = make(60, 50, 40, BF, 3)
    compare(ids.view(3, 4, 5), w, dy.view(3, 4, 5, 40), cast=lambda i: i.int())
    wide = torch.randn(50, 91, device=DEV).to(BF)
    compare(ids, wide[:, 3:43], dy)                              # rows off 16-byte boundaries
    compare(ids, wide[:, :40], dy.repeat(1, 2)[:, 40:])
    compare(ids, torch.randn(40, 50, device=DEV).to(BF).t(), dy)
    compare(ids.repeat(2)[::2], w, dy[:1].expand(60, 40))       # one row of dy for all


def test_no_tokens():
    ids, w, _ = make(1, 5, 8, F32)
    w.requires_grad_(True)
    y = tt.embedding(ids[:0], w)
    assert y.shape == (0, 8)
    y.sum().backward()
    assert not w.grad.any()


def test_ids_outside_the_table():
    ids, w, dy = make(100, 30, 24, F16, 4)
    bad = ids.clone()
    bad[7], bad[50] = -1, 30
    w.requires_grad_(True)
    y = tt.embedding(bad, w)
    y.backward(dy)
    assert y[7].isnan().all() and y[50].isnan().all()
    with pytest.raises(tt.TTError):
        tt.check_device_status()
    tt.check_device_status()
    keep = torch.ones(100, dtype=torch.bool, device=DEV)
    keep[7] = keep[50] = False
    want = torch.zeros(30, 24, dtype=torch.float64, device=DEV).index_add_(
        0, ids[keep], dy[keep].double())
    check("dw", w.grad, want, torch.zeros_like(want).index_add_(
        0, ids[keep], dy[keep].double().abs()), 100)


def test_same_bits_every_time():
    ids, w, dy = make(8000, 500, 264, BF, 5, 0.3)
    w.requires_grad_(True)
    runs = []
    for _ in range(3):
        dw, = torch.autograd.grad(tt.embedding(ids, w), w, dy)
        runs.append(dw)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_captured_and_replayed():
    ids, w, dy = make(300, 400, 64, BF, 6)
    w.requires_grad_(True)
    step = lambda: torch.autograd.grad(tt.embedding(ids, w, scale=2.0), w, dy)[0]
    step()
    graph, pool = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        dw = step()
    ids.copy_(make(300, 400, 64, BF, 7)[0])
    graph.replay()
    want = torch.zeros(400, 64, dtype=torch.float64, device=DEV).index_add_(0, ids, 2 * dy.double())
    check("dw", dw, want, torch.zeros_like(want).index_add_(0, ids, 2 * dy.double().abs()), 50)


def test_on_another_stream():
    ids, w, dy = make(500, 60, 128, F32, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        compare(ids, w, dy)
    torch.cuda.current_stream().wait_stream(side)


def test_refusals():
    ids, w, dy = make(4, 5, 8, F32)
    with pytest.raises(TypeError):
        tt.embedding(ids.float(), w)
    with pytest.raises(TypeError):
        tt.embedding(ids, w.double())
    with pytest.raises(RuntimeError):
        tt.embedding(ids.cpu(), w)
    for bad in (dict(padding_idx=5), dict(padding_idx=-6), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            tt.embedding(ids, w, **bad)
    with pytest.raises(ValueError):
        tt.embedding(ids, w[0])
    w.requires_grad_(True)
    g, = torch.autograd.grad(tt.embedding(ids, w).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_the_widest_row_and_wider_ones():
    H = 1 << 22
    w = torch.randn(2, H, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    ids = torch.tensor([1, 1, 0], device="cuda")
    y = tt.embedding(ids, w)
    assert torch.equal(y, w[ids])
    dw, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(dw, torch.tensor([[1.], [2.]], device="cuda").bfloat16().expand(2, H))
    tt.check_device_status()
    with pytest.raises(ValueError):
        tt.embedding(ids, torch.zeros(2, H + 1, device="cuda", dtype=torch.bfloat16))
