"""``apply_rotary`` against the definition in 64 bits: both pair layouts, part
of the head, odd sizes, strides, q alone, and its gradient.

Bounds: an output is a cos - b sin: three fp32 roundings over |a cos| + |b sin|,
then one rounding to the output's type; steps = 4.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import check, directional

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def turned(x, pos, table, interleaved, sign=1.0):
    """(result, magnitude) in 64 bits, pair by pair."""
    x, t = x.double(), table.double()[pos.long()]
    R = t.shape[1]
    h = R // 2
    c, s = t[:, None, :h], sign * t[:, None, h:]
    first = torch.arange(h, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else h)
    a, b = x[..., first], x[..., second]
    y, m = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    m[..., first] = (a * c).abs() + (b * s).abs()
    m[..., second] = (b * c).abs() + (a * s).abs()
    return y, m


def data(N, hq, hk, D, R, dtype, P=513, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(N, hq, D, generator=g, device=DEV).to(dtype)
    k = torch.randn(N, hk, D, generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, P, (N,), generator=g, device=DEV)
    return q, k, pos, tt.rotary_table(P, R, 1e4, device=DEV)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,hq,hk,D,R,dtype", [
    (1, 1, 1, 2, 2, torch.float32), (1, 32, 8, 128, 128, torch.bfloat16),
    (47, 4, 2, 64, 64, torch.float32), (333, 16, 2, 256, 64, torch.float16),
    (130, 5, 1, 80, 80, torch.bfloat16), (65, 3, 3, 96, 36, torch.bfloat16),
    (65, 3, 1, 67, 22, torch.float16), (9, 2, 1, 7, 6, torch.float32),
    (1000, 32, 8, 128, 128, torch.bfloat16), (12, 1, 1, 1030, 516, torch.float32),
    (3, 40, 9, 64, 2, torch.bfloat16),
])
def test_both_directions(N, hq, hk, D, R, dtype, interleaved):
    q, k, pos, table = data(N, hq, hk, D, R, dtype)
    q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = tt.apply_rotary(q, k, pos, table, interleaved=interleaved)
    g = torch.Generator(device=DEV).manual_seed(1)
    dq = torch.randn(q.shape, generator=g, device=DEV).to(dtype)
    dk = torch.randn(k.shape, generator=g, device=DEV).to(dtype)
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    for name, got, x, sign in (("q", qo, q, 1.0), ("k", ko, k, 1.0), ("dq", gq, dq, -1.0),
                               ("dk", gk, dk, -1.0)):
        assert got.dtype == dtype and got.is_contiguous()
        check(name, got.detach(), *turned(x.detach(), pos, table, interleaved, sign), 4)
    tt.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_positions_types(dtype):
    q, k, pos, table = data(77, 4, 2, 64, 32, dtype)
    want = tt.apply_rotary(q, k, pos, table)
    g = torch.Generator(device=DEV).manual_seed(2)
    # views of a packed projection, one of them off by a single element
    for lead in (0, 1, 4):
        buf = torch.randn(77, lead + 8 * 64, generator=g, device=DEV).to(dtype)
        buf[:, lead:lead + 256] = q.view(77, 256)
        buf[:, lead + 256:lead + 384] = k.view(77, 128)
        got = tt.apply_rotary(buf[:, lead:lead + 256].view(77, 4, 64),
                              buf[:, lead + 256:lead + 384].view(77, 2, 64), pos.int(), table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # head-major storage, an inner stride, shared (expanded) heads, strided positions
    got = tt.apply_rotary(q.transpose(0, 1).contiguous().transpose(0, 1),
                          k.transpose(1, 2).contiguous().transpose(1, 2),
                          pos.repeat_interleave(2)[::2], table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = k[:, :1].expand(-1, 5, -1)
    assert torch.equal(tt.apply_rotary(q, one, pos, table)[1],
                       tt.apply_rotary(q, one.contiguous(), pos, table)[1])
    alone, none = tt.apply_rotary(q, None, pos, table)
    assert none is None and torch.equal(alone, want[0])


def test_gradient_by_differences():
    # linear in q and k: the central difference is exact up to rounding, about
    # 2^-24 sqrt(n) |x| / h of a value; 1e-3 is far above it
    q, k, pos, table = data(20, 3, 2, 32, 24, torch.float32)
    ws = [torch.randn_like(q), torch.randn_like(k)]
    q.requires_grad_(True), k.requires_grad_(True)
    grads = torch.autograd.grad(tt.apply_rotary(q, k, pos, table), [q, k], ws)
    directional(lambda a, b: tt.apply_rotary(a, b, pos, table), [q, k], ws, grads, 0.5, 1e-3)


def test_gradient_of_one_output_and_of_shared_heads():
    q, k, pos, table = data(20, 3, 1, 32, 32, torch.float32)
    k.requires_grad_(True)
    out = tt.apply_rotary(q, k.expand(-1, 4, -1), pos, table)[1]
    w = torch.randn_like(out)
    gk, = torch.autograd.grad(out, [k], [w])
    y, m = turned(w, pos, table, False, -1.0)
    check("dk", gk, y.sum(1, keepdim=True), m.sum(1, keepdim=True), 8)


def test_no_tokens():
    q, k, pos, table = data(0, 4, 2, 64, 64, torch.bfloat16)
    qo, ko = tt.apply_rotary(q, k, pos, table)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)


@pytest.mark.parametrize("bad", [-1, 513, 1 << 40])
def test_position_outside_the_table_is_reported(bad):
    q, k, pos, table = data(5, 2, 1, 16, 8, torch.float32)
    want = tt.apply_rotary(q, k, pos, table)[0]
    pos[3] = bad
    got = tt.apply_rotary(q, k, pos, table)[0]
    keep = [0, 1, 2, 4]
    assert torch.equal(got[keep], want[keep])
    assert got[3, :, :8].isnan().all() and torch.equal(got[3, :, 8:], q[3, :, 8:])
    with pytest.raises(tt.TTError):
        tt.check_device_status(DEV)
    tt.check_device_status(DEV)


def test_another_stream():
    q, k, pos, table = data(500, 8, 2, 64, 64, torch.bfloat16)
    want = tt.apply_rotary(q, k, pos, table)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = tt.apply_rotary(q, k, pos, table)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    q, k, pos, table = data(5, 2, 1, 16, 8, torch.float32)
    with pytest.raises(RuntimeError):
        tt.apply_rotary(q.cpu(), k, pos, table)
    with pytest.raises(RuntimeError):
        tt.apply_rotary(q, k, pos.cpu(), table)
    with pytest.raises(TypeError):
        tt.apply_rotary(q.double(), k.double(), pos, table)
    with pytest.raises(TypeError):
        tt.apply_rotary(q, k.bfloat16(), pos, table)
    with pytest.raises(TypeError):
        tt.apply_rotary(q, k, pos.float(), table)
    with pytest.raises(TypeError):
        tt.apply_rotary(q, k, pos, table.bfloat16())
    for a in ((q[0], k, pos, table), (q, k[:4], pos, table), (q, k[..., :8], pos, table),
              (q, k, pos[:4], table), (q, k, pos[None], table), (q[:, :0], k, pos, table),
              (q, k, pos, table[:, :7]), (q, k, pos, tt.rotary_table(9, 18, device=DEV))):
        with pytest.raises(ValueError):
            tt.apply_rotary(*a)


def test_differentiating_twice_is_refused():
    q, k, pos, table = data(5, 2, 1, 16, 8, torch.float32)
    q.requires_grad_(True)
    g, = torch.autograd.grad(tt.apply_rotary(q, k, pos, table)[0].sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [q])


def test_offsets_over_32_bits():
    # 2^31 elements and more, read through a strided view
    N, H, D = (1 << 17) + 3, 128, 128
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.zeros(N, H, D, dtype=torch.bfloat16, device=DEV)
    rows = [0, (1 << 17) - 1, 1 << 17, N - 1]
    q[rows] = torch.randn(4, H, D, generator=g, device=DEV).to(q.dtype)
    pos = torch.randint(0, 513, (N,), generator=g, device=DEV)
    table = tt.rotary_table(513, D, 1e4, device=DEV)
    got, _ = tt.apply_rotary(q, None, pos, table)
    check("q", got[rows], *turned(q[rows], pos[rows], table, False), 4)
    k = q.transpose(0, 1).contiguous().transpose(0, 1)          # head-major storage
    assert torch.equal(tt.apply_rotary(k, None, pos, table)[0][rows], got[rows])
