"""A module that ``fuse_gated_mlps`` has taken and that changes afterwards: adapters,
hooks, other parts.  The kernel's place is taken by plain products, which count their
calls (what the kernel computes needs a GPU).
"""
import copy
import sys

import pytest
import torch
from torch import nn

import tree_training_b200 as tt

MODULE = sys.modules["tree_training_b200.gated_linear"]


class Mlp(nn.Module):
    def __init__(self, hidden=32, features=48):
        super().__init__()
        self.gate_proj = nn.Linear(hidden, features, bias=False)
        self.up_proj = nn.Linear(hidden, features, bias=False)
        self.down_proj = nn.Linear(features, hidden, bias=False)
        self.act_fn = nn.SiLU()

    def forward(self, hidden):
        return self.down_proj(self.act_fn(self.gate_proj(hidden)) * self.up_proj(hidden))


class Adapter(nn.Module):
    """A low-rank term beside a projection, whose weight it shows as its own."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.low = nn.Linear(base.in_features, 4, bias=False)
        self.high = nn.Linear(4, base.out_features, bias=False)

    @property
    def weight(self):
        return self.base.weight

    @property
    def bias(self):
        return self.base.bias

    def forward(self, x):
        return self.base(x) + self.high(self.low(x))


@pytest.fixture
def kernel(monkeypatch):
    calls = []

    def stand_in(x, w_gate, w_up, activation="silu"):
        calls.append((x.dtype, w_gate.dtype, activation))
        return getattr(nn.functional, activation)(x @ w_gate.t()) * (x @ w_up.t())
    monkeypatch.setattr(MODULE, "gated_linear", stand_in)
    return calls


def fused(seed=0):
    torch.manual_seed(seed)
    mod = Mlp()
    own = copy.deepcopy(mod)
    assert tt.fuse_gated_mlps(nn.ModuleList([mod])) == 1
    return mod, own


def same(mod, own, x, rtol=1e-5):
    torch.testing.assert_close(mod(x), own(x), rtol=rtol, atol=1e-6)


def test_a_taken_module_calls_the_kernel(kernel):
    mod, own = fused()
    same(mod, own, torch.randn(5, 32))
    assert kernel == [(torch.float32, torch.float32, "silu")]
    mod.down_proj = Adapter(mod.down_proj)          # (that one is called as it is)
    mod.down_proj.base.register_forward_hook(lambda *a: None)
    mod(torch.randn(5, 32))
    assert len(kernel) == 2


@pytest.mark.parametrize("name", ["gate_proj", "up_proj"])
def test_an_adapter_put_over_a_projection(kernel, name):
    mod, own = fused()
    for m in (mod, own):
        torch.manual_seed(1)
        setattr(m, name, Adapter(getattr(m, name)))
    x = torch.randn(5, 32)
    same(mod, own, x)
    mod(x).sum().backward()
    own(x).sum().backward()
    for a, b in zip(mod.parameters(), own.parameters()):
        assert a.grad is not None and b.grad is not None
        torch.testing.assert_close(a.grad, b.grad)
    assert not kernel
    setattr(mod, name, getattr(mod, name).base)     # taken off again
    mod(x)
    assert len(kernel) == 1


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "act_fn"])
@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre"])
def test_a_hook_registered_later(kernel, name, kind):
    mod, _ = fused()
    seen = []
    handle = getattr(getattr(mod, name), f"register_{kind}_hook")(lambda *a: seen.append(name))
    x = torch.randn(5, 32, requires_grad=True)
    mod(x).sum().backward()
    assert seen == [name] and not kernel
    handle.remove()
    mod(x)
    assert seen == [name] and len(kernel) == 1


def test_hooks_of_all_modules(kernel):
    mod, own = fused()
    seen = []
    handle = nn.modules.module.register_module_forward_hook(lambda m, *a: seen.append(m))
    try:
        same(mod, own, torch.randn(5, 32))
    finally:
        handle.remove()
    assert mod.gate_proj in seen and mod.act_fn in seen and not kernel


def test_parts_that_are_replaced(kernel):
    x = torch.randn(5, 32)

    def other(change):
        mod, own = fused()
        for m in (mod, own):
            torch.manual_seed(2)
            change(m)
        same(mod, own, x)
        assert not kernel
    other(lambda m: setattr(m, "gate_proj", nn.Linear(32, 48)))
    other(lambda m: setattr(m, "act_fn", nn.Tanh()))
    other(lambda m: setattr(m.gate_proj, "bias", nn.Parameter(torch.randn(48))))
    other(lambda m: nn.utils.parametrizations.weight_norm(m.up_proj))
    other(lambda m: setattr(m.up_proj, "forward", lambda t: t.new_ones(t.shape[0], 48)))
    mod, own = fused()                              # (a new weight of the same kind is used)
    for m in (mod, own):
        torch.manual_seed(3)
        m.gate_proj = nn.Linear(32, 48, bias=False)
        m.act_fn = nn.GELU()
    same(mod, own, x)
    assert [k[2] for k in kernel] == ["gelu"]


def test_a_class_whose_forward_is_replaced(kernel):
    mod, _ = fused()
    before = Mlp.forward
    try:
        Mlp.forward = lambda self, hidden: hidden * 2
        x = torch.randn(5, 32)
        assert torch.equal(mod(x), x * 2) and not kernel
    finally:
        Mlp.forward = before


def test_other_ways_to_call(kernel):
    mod, own = fused()
    x = torch.randn(5, 32)
    torch.testing.assert_close(mod(hidden=x), own(hidden=x))
    with pytest.raises(TypeError):
        mod(x, 1)
    with pytest.raises(TypeError):
        mod()


def test_copies_are_of_their_own_parts(kernel):
    mod, _ = fused()
    other = copy.deepcopy(mod)
    with torch.no_grad():
        other.gate_proj.weight.zero_()
    x = torch.randn(5, 32)
    assert not other(x).any() and mod(x).any() and len(kernel) == 2


@pytest.mark.parametrize("given", [torch.float32, torch.bfloat16])
def test_under_autocast(kernel, given):
    """In autocast's type, as the projections of the module's own forward."""
    mod, own = fused()
    x = torch.randn(5, 32)
    grads = []
    for m in (mod, own):
        leaf = x.to(given).requires_grad_(True)
        with torch.autocast("cpu", torch.bfloat16):
            y = m(leaf)
        assert y.dtype == torch.bfloat16
        grads.append([y, *torch.autograd.grad(y.float().square().sum(), [leaf, *m.parameters()])])
    assert kernel == [(torch.bfloat16, torch.bfloat16, "silu")]
    for a, b in zip(*grads):
        assert a.dtype == b.dtype
        assert float((a - b).norm()) <= 2.0 ** -6 * float(b.norm())      # a few roundings to bf16
    with torch.autocast("cpu", torch.bfloat16, enabled=False):
        mod(x)
    assert kernel[1:] == [(torch.float32, torch.float32, "silu")]
