"""The activations far from 0, of single products: what is small there is kept as far as
the type holds it, and what is large has slope 1.

Bounds.  The exponential of an argument z errs by (2 + 1.2 |z|) units of fp32, the
argument itself (tanh's) by a few of its own: 2^-23 (8 + 8 |z|) of the value altogether,
beside one rounding of each gradient of a product and one of the result.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import TINY, UNIT
from tests.test_gated_linear_gpu import act64

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def products(g, T, dtype):
    """x [T, 16], wg and wu [F, 16] with x wg^T = g in every row, x wu^T = 1."""
    x = torch.zeros(T, 16, device=DEV)
    wg, wu = (torch.zeros(len(g), 16, device=DEV) for _ in range(2))
    x[:, 0] = x[:, 1] = 1
    wg[:, 0], wu[:, 1] = g, 1
    return [t.to(dtype).requires_grad_(True) for t in (x, wg, wu)]


def run(g, T, dtype, act):
    leaves = products(g, T, dtype)
    h = tt.gated_linear(*leaves, activation=act)
    # dwg[f, 0] and dwu[f, 1]: the sums over the rows of dg = act'(g) and du = act(g)
    _, dwg, dwu = torch.autograd.grad(h, leaves, torch.eye(T, len(g), device=DEV).to(dtype))
    tt.check_device_status()
    g = leaves[1][:, 0].detach().double().requires_grad_(True)
    a = act64(g, act)
    d, = torch.autograd.grad(a.sum(), g)
    n = min(T, len(g))
    return g.detach(), a.detach(), d, h.detach(), dwg[:n, 0], dwu[:n, 1]


@pytest.mark.parametrize("T", [1, 200])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_far_below_zero(dtype, T):
    g = torch.arange(-103.5, -60, 0.25, device=DEV)
    g, a, d, h, dwg, dwu = run(g, T, dtype, "silu")
    rel = UNIT[dtype] + 2.0 ** -23 * (8 + 8 * g.abs())
    # (fp32's own subnormals on the way: exp(-103) is one unit of them, and g times it)
    tiny = TINY[dtype] + 2.0 ** -149 * (2 + g.abs())
    n = len(dwg)
    assert ((h.double() - a).abs() <= rel * a.abs() + tiny).all()
    assert ((dwu.double() - a[:n]).abs() <= 2 * (rel * a.abs() + tiny)[:n]).all()
    assert ((dwg.double() - d[:n]).abs() <= 2 * (rel * (1 + g.abs()) * g.exp() + tiny)[:n]).all()
    assert (h[:, g > -87] != 0).all() and (dwu[g[:n] > -87] != 0).all()


@pytest.mark.parametrize("T", [1, 200])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_very_large_products(act, dtype, T):
    sizes = torch.logspace(3, 37, 100, device=DEV).to(dtype).float()
    g, a, d, h, dwg, dwu = run(torch.cat([sizes, -sizes]), T, dtype, act)
    want = g.clamp(min=0)
    n = len(dwg)
    assert torch.equal(h.double(), want.expand_as(h))
    assert torch.equal(dwu.double(), want[:n])
    assert torch.equal(dwg.double(), (g[:n] > 0).double())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_nan_has_no_slope(act, dtype):
    leaves = products(torch.tensor([1.0, float("nan"), 2.0], device=DEV), 130, dtype)
    h = tt.gated_linear(*leaves, activation=act)
    _, dwg, dwu = torch.autograd.grad(h, leaves, torch.ones_like(h))
    assert h[:, 1].isnan().all() and dwg[1, 0].isnan() and dwu[1, 1].isnan()
    assert h[:, ::2].isfinite().all() and dwg[::2, 0].isfinite().all()
