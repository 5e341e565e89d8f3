"""The layer operators have no forward-mode derivatives: an input that carries a
tangent is refused, whether or not it also wants a gradient, instead of giving a
result without one."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def calls():
    """name -> (a call of tensors, the tensors that may carry a tangent)"""
    n = lambda *s: torch.randn(*s, device=DEV)
    pos, tok = torch.arange(4, device=DEV), torch.arange(4, device=DEV)
    plan = tt.expert_plan(torch.tensor([[0, 1]] * 4, device=DEV), 2)
    return {
        "logits": (lambda x: tt.token_logprobs(x, tok, top_k=2), [n(4, 32)]),
        "rotary": (lambda q, k, t: tt.apply_rotary(q, k, pos, t),
                   [n(4, 2, 8), n(4, 1, 8), tt.rotary_table(8, 8, device=DEV)]),
        "norm": (lambda x, r, w, p, g: tt.residual_norm(x, r, w, post_weight=p, gate=g),
                 [n(4, 16), n(4, 16), n(16), n(16), n(4, 16)]),
        "dispatch": (lambda x: tt.expert_dispatch(x, plan), [n(4, 8)]),
        "combine": (lambda ys, w: tt.expert_combine(ys, w, plan), [n(8, 8), n(4, 2)]),
    }


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("wants_gradient", [False, True])
@pytest.mark.parametrize("name", ["logits", "rotary", "norm", "dispatch", "combine"])
def test_tangents_are_refused(name, wants_gradient, no_grad):
    f, xs = calls()[name]
    for i in range(len(xs)):
        with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
            args = [x.detach().requires_grad_(wants_gradient) for x in xs]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError):
                f(*args)
        f(*xs)                              # without one the call goes through


@pytest.mark.parametrize("name", ["logits", "rotary", "norm", "dispatch", "combine"])
def test_function_transforms_are_refused(name):
    f, xs = calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: f(x, *xs[1:])[0], (xs[0],), (torch.ones_like(xs[0]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: f(x, *xs[1:])[0])(torch.stack([xs[0], xs[0]]))


@pytest.mark.parametrize("name", ["logits", "rotary", "norm", "dispatch", "combine"])
def test_gradients_that_carry_a_tangent_are_refused(name):
    f, xs = calls()[name]
    x = xs[0].requires_grad_(True)
    y = f(*xs)
    y = y if isinstance(y, torch.Tensor) else y[0]
    with fwd.dual_level():
        g = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, [x], [g], retain_graph=True)
    torch.autograd.grad(y, [x], [torch.ones_like(y)])
