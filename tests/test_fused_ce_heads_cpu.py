"""The fused losses of ``tree_grad_hybrid`` go by the LM head's weight alone: heads that
do more are refused, not computed without it."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

from tree_training_b200.hybrid import make_tree_loss_fn, tree_grad_hybrid


class Reached(Exception):
    """The arguments were accepted."""


class Model(nn.Module):
    def __init__(self, head, **config):
        super().__init__()
        self.model, self.lm_head = nn.Identity(), head
        self._config = SimpleNamespace(**config)
        self.asked = 0

    @property
    def config(self):
        return self._config

    def parameters(self, recurse=True):
        raise Reached


class Adapter(nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base, self.bias = base, None
        self.more = nn.Linear(8, 20, bias=False)

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + self.more(x)


def step(model, fused_ce):
    tree_grad_hybrid(model, [], make_tree_loss_fn([], [], 1), 100, fused_ce=fused_ce)


def hooked(head):
    head.register_forward_hook(lambda *a: None)
    return head


def replaced(head):
    head.forward = lambda x: x
    return head


@pytest.mark.parametrize("fused_ce", [True, "pieces"])
def test_heads(fused_ce, monkeypatch):
    monkeypatch.setattr("tree_training_b200.hybrid._ensure_tree_attention", lambda model: None)
    plain = lambda: nn.Linear(8, 20, bias=False)
    for model in (Model(nn.Linear(8, 20)), Model(Adapter(plain())), Model(hooked(plain())),
                  Model(replaced(plain())), Model(plain(), final_logit_softcapping=30.0),
                  Model(plain(), logit_scale=0.0625), Model(plain(), logits_scaling=8.0)):
        with pytest.raises(ValueError):
            step(model, fused_ce)
        with pytest.raises(Reached):
            step(model, False)
    for model in (Model(plain()), Model(plain(), final_logit_softcapping=None, logit_scale=1.0)):
        with pytest.raises(Reached):
            step(model, fused_ce)
    with pytest.raises(ValueError):
        step(SimpleNamespace(lm_head=plain()), fused_ce)
