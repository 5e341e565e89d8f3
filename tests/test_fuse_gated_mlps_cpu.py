"""Which modules ``fuse_gated_mlps`` takes: those whose forward is
down(act(gate(x)) * up(x)) and nothing else, whatever the values that it would change.
(What a taken module computes needs a GPU.)
"""
import pytest
import torch
from torch import nn
from torch.nn import functional as F

import tree_training_b200 as tt


class Mlp(nn.Module):
    def __init__(self, act=None, hidden=32, features=48):
        super().__init__()
        self.gate_proj = nn.Linear(hidden, features, bias=False)
        self.up_proj = nn.Linear(hidden, features, bias=False)
        self.down_proj = nn.Linear(features, hidden, bias=False)
        self.act_fn = act or nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


def taken(mod):
    return tt.fuse_gated_mlps(nn.ModuleList([mod]))


class Clamped(Mlp):
    limit = 7.0

    def forward(self, x):
        g = self.gate_proj(x).clamp(max=self.limit)
        u = self.up_proj(x).clamp(-self.limit, self.limit)
        return self.down_proj(self.act_fn(g) * u)


@pytest.mark.parametrize("limit", [4.0, 7.0, 10.0, 1e4])
def test_a_bound_that_few_values_reach(limit):
    torch.manual_seed(0)
    mod = Clamped(hidden=256, features=512)
    mod.limit = limit
    for p in mod.parameters():
        nn.init.normal_(p, std=0.02)
    x = torch.randn(3, 256) * 50 * limit
    want = mod(x)
    assert taken(mod) == 0
    assert torch.equal(mod(x), want)


def test_dropout_before_a_projection_of_zeros():
    class Dropping(Mlp):
        def forward(self, x):
            h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
            return self.down_proj(F.dropout(h, 0.1, self.training))
    mod = Dropping()
    nn.init.zeros_(mod.down_proj.weight)
    assert taken(mod) == 0


def test_what_is_done_only_in_training_or_only_outside_it():
    class Noisy(Mlp):
        when = True

        def forward(self, x):
            h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
            return self.down_proj(h * 1.0 if self.training is self.when else h)
    for when in (True, False):
        mod = Noisy()
        mod.when = when
        assert taken(mod) == 0


def test_other_orders_of_the_same_and_other_uses_of_the_parts():
    class Turned(Mlp):
        def forward(self, x):
            u = self.up_proj(x)
            return self.down_proj(u * self.act_fn(self.gate_proj(x)))

    class Swapped(Mlp):                       # up through the activation
        def forward(self, x):
            return self.down_proj(self.gate_proj(x) * self.act_fn(self.up_proj(x)))

    class Twice(Mlp):
        def forward(self, x):
            return self.down_proj(self.act_fn(self.act_fn(self.gate_proj(x))) * self.up_proj(x))

    class Residual(Mlp):
        def forward(self, x):
            return x + super().forward(x)

    class Scaled(Mlp):
        def forward(self, x):
            return super().forward(x) * 1.0

    class Squared(Mlp):
        def forward(self, x):
            g = self.act_fn(self.gate_proj(x))
            self.up_proj(x)
            return self.down_proj(g * g)
    assert taken(Turned()) == 1
    for form in (Swapped, Twice, Residual, Scaled, Squared):
        assert taken(form()) == 0, form


def test_forwards_of_other_arguments_or_results():
    class Asking(Mlp):
        def forward(self, x, layer):
            return super().forward(x)

    class Telling(Mlp):
        def forward(self, x):
            return super().forward(x), None

    class Raising(Mlp):
        def forward(self, x):
            raise NotImplementedError
    for form in (Asking, Telling, Raising):
        assert taken(form()) == 0, form


def test_activations_that_only_share_a_name():
    class SiLU(nn.Module):
        def forward(self, x):
            return F.silu(x).clamp(max=5.0)

    class GELU(nn.GELU):
        def forward(self, x):
            return super().forward(x) * 2
    watched = nn.SiLU()
    seen = []
    watched.register_forward_hook(lambda *a: seen.append(1))
    replaced = nn.SiLU()
    replaced.forward = lambda x: x
    for act in (SiLU(), GELU(), watched, replaced):
        assert taken(Mlp(act)) == 0, act
    assert not seen
    for act in (nn.SiLU(), nn.GELU(), nn.GELU(approximate="tanh"), nn.ReLU()):
        assert taken(Mlp(act)) == 1, act


@pytest.mark.parametrize("name", ["silu", "swish", "gelu", "gelu_python", "gelu_pytorch_tanh",
                                  "gelu_python_tanh", "relu"])
def test_activations_of_hf_models(name):
    activations = pytest.importorskip("transformers.activations")
    assert taken(Mlp(activations.ACT2FN[name])) == 1
    assert taken(Mlp(activations.ACT2FN["gelu_new"])) == 0


def test_parts_of_other_kinds():
    class Wide(nn.Linear):
        def forward(self, x):
            return super().forward(x) * 2
    for name in ("gate_proj", "up_proj", "down_proj"):
        mod = Mlp()
        old = getattr(mod, name)
        setattr(mod, name, Wide(old.in_features, old.out_features, bias=False))
        assert taken(mod) == 0
        mod = Mlp()
        getattr(mod, name).forward = lambda x: x
        assert taken(mod) == 0
    mod = Mlp()
    mod.up_proj.double()
    assert taken(mod) == 0


def test_models_without_data():
    with torch.device("meta"):
        assert taken(Mlp()) == 1
        assert taken(Clamped()) == 0


def test_state_is_left_as_it_was():
    class Dropping(Mlp):
        def forward(self, x):
            return F.dropout(super().forward(x), 0.5, self.training)
    m = nn.ModuleList([Mlp(), Dropping(), Clamped()]).eval()
    state = torch.get_rng_state()
    assert tt.fuse_gated_mlps(m) == 1
    assert torch.equal(torch.get_rng_state(), state)
    assert not any(b.training for b in m.modules())
    assert not any(b._forward_hooks or b._forward_pre_hooks for b in m.modules())
    assert all(p.grad is None for p in m.parameters())
    assert tt.fuse_gated_mlps(m) == 0


@pytest.mark.parametrize("enabled", [False, True])
@pytest.mark.filterwarnings("ignore:.*CUDA is not available")
def test_forwards_that_set_autocast_themselves(enabled):
    class Setting(Mlp):
        def forward(self, x):
            with torch.autocast("cuda", torch.bfloat16, enabled=enabled):
                return super().forward(x)

    class Frozen(Mlp):
        def forward(self, x):
            with torch.no_grad():
                g = self.gate_proj(x)
            return self.down_proj(self.act_fn(g) * self.up_proj(x))
    before = torch.is_autocast_enabled("cuda")
    assert taken(Setting()) == 0
    assert taken(Frozen()) == 0
    assert torch.is_autocast_enabled("cuda") == before
