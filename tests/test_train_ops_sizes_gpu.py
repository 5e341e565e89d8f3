"""The training operators where offsets pass 32 bits, and where a kernel's grid would."""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_embedding_table_over_2_to_the_32_bytes():
    V, H = 70001, 40000                          # 2.8e9 elements
    w = torch.zeros(V, H, dtype=torch.float16, device=DEV)
    w[-1], w[V // 2] = 3.0, -2.0
    w.requires_grad_(True)
    ids = torch.tensor([V - 1, 0, V // 2, V - 1], device=DEV)
    y = tt.embedding(ids, w)
    assert y[:, ::1999].tolist() == [[v] * 21 for v in (3.0, 0.0, -2.0, 3.0)]
    dy = torch.arange(1, 5, device=DEV, dtype=torch.float16)[:, None].expand(4, H)
    dw, = torch.autograd.grad(y, w, dy)
    assert (dw[-1] == 5).all() and (dw[0] == 2).all() and (dw[V // 2] == 3).all()
    assert not dw[1:V // 2].any() and not dw[V // 2 + 1:-1].any()


def test_gated_linear_results_over_2_to_the_32_bytes():
    T, H, F = 300001, 8, 8192                    # 2.5e9 elements
    x = torch.ones(T, H, dtype=torch.bfloat16, device=DEV)
    x[-1] = 2.0
    w = torch.full((F, H), 0.125, dtype=torch.bfloat16, device=DEV)
    h = tt.gated_linear(x, w, w, activation="relu")
    assert (h[0] == 1).all() and (h[T // 2] == 1).all() and (h[-1] == 4).all()
    tt.check_device_status()


def test_gated_linear_of_many_fp32_rows():
    T = 4500000                                  # over 65,535 tiles of 64
    x = torch.ones(T, 4, device=DEV)
    x[-1] = 2.0
    w = torch.full((4, 4), 0.25, device=DEV)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    h = tt.gated_linear(x, w, w, activation="relu")
    assert h[0].tolist() == [1.0] * 4 and h[-1].tolist() == [4.0] * 4
    dx, _ = torch.autograd.grad(h, leaves, torch.ones_like(h))
    assert dx[0].tolist() == [2.0] * 4 and dx[-1].tolist() == [4.0] * 4


def test_linear_ce_weight_over_2_to_the_32_bytes():
    V, H = 600007, 4096                          # 2.5e9 elements
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=DEV)
    w[-1, 0] = 4.0
    x = torch.zeros(3, H, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = torch.tensor([1.0, 0.0, 2.0])
    r = tt.linear_cross_entropy(x, w, torch.tensor([V - 1, 5, V - 1], device=DEV))
    z = torch.tensor([4.0, 0.0, 8.0], dtype=torch.float64)
    lse = torch.log(torch.exp(z) + V - 1)
    want = lse - torch.tensor([4.0, 0.0, 8.0], dtype=torch.float64)
    # the sum of V exponentials in fp32, by tiles
    assert ((r.losses.double().cpu() - want).abs() <= 64 * 2.0 ** -24 * lse).all()
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(tt.linear_cross_entropy(x, w, torch.tensor(
        [V - 1, 5, V - 1], device=DEV)).losses.sum(), [x, w])
    p = torch.exp(z - lse)                       # of the last word
    got = dw[-1, 0].double().cpu()
    want = (p[0] - 1) * 1 + p[1] * 0 + (p[2] - 1) * 2
    assert abs(float(got - want)) <= 3 * 2.0 ** -8 * abs(float(want))
    assert not dw[:, 1:].any()


def test_gradients_over_2_to_the_31_elements():
    t = torch.zeros((1 << 31) + 7, dtype=torch.bfloat16, device=DEV)
    t[0], t[-1], t[1 << 31] = 3.0, 4.0, 12.0
    assert float(tt.grad_norm([t])) == 13.0
    assert float(tt.clip_grad_norm([t], 6.5, eps=0.0)) == 13.0
    assert (t[0], t[-1], t[1 << 31]) == (1.5, 2.0, 6.0)
