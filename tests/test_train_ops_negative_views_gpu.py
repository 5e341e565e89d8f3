"""Tensors that keep their sign beside their memory (the imaginary part of a conjugate):
their values count, not what stands in memory.  Products of negated inputs are the
negated products, bit for bit.
"""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tensor(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def test_the_imaginary_part_of_a_conjugate():
    z = torch.complex(tensor(6, 16), tensor(6, 16, seed=1))
    x = z.conj().imag
    assert x.is_neg()
    w = tensor(24, 16, seed=2), tensor(24, 16, seed=3)
    assert torch.equal(tt.gated_linear(x, *w), tt.gated_linear(-z.imag, *w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_inputs_and_gradients(dtype):
    neg = torch._neg_view
    ids = torch.randint(0, 40, (7, 9), device=DEV)
    x, table = tensor(50, 32, dtype=dtype), tensor(40, 32, seed=1, dtype=dtype)
    wg, wu = tensor(48, 32, seed=2, dtype=dtype), tensor(48, 32, seed=3, dtype=dtype)
    labels = torch.randint(0, 40, (50,), device=DEV)
    for f, args in ((lambda w: tt.embedding(ids, w), (table,)),
                    (tt.gated_linear, (x, wg, wu)),
                    (lambda a, w: tt.linear_cross_entropy(a, w, labels).losses, (x, table))):
        plain = [(-a).requires_grad_(True) for a in args]
        views = [neg(a).requires_grad_(True) for a in args]
        y, v = f(*plain), f(*views)
        assert torch.equal(y, v)
        dy = tensor(*y.shape, seed=5, dtype=y.dtype)
        want = torch.autograd.grad(y, plain, -dy)
        got = torch.autograd.grad(v, views, neg(dy))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    tt.check_device_status()


def test_norms_and_clipping():
    a, b = tensor(1000), tensor(33, 5, seed=1)
    for p in (1.0, 2.0, float("inf")):
        assert torch.equal(tt.grad_norm([torch._neg_view(a), b], p), tt.grad_norm([a, b], p))
    with pytest.raises(ValueError):
        tt.clip_grad_norm([torch._neg_view(a), b], 1.0)
    with pytest.raises(ValueError):
        tt.clip_grad_norm([a, b], 1.0, out=[torch._neg_view(a.clone()), b.clone()])
