"""``expert_dispatch`` / ``expert_combine`` with plans that the caller made or
changed: other strides, and slots and offsets outside the sorted rows, which drop
their choices.  Every copy and sum here is exact."""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1


def everything(plan, T, k, H, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    n = lambda *s: torch.randint(-3, 4, s, generator=g, device=DEV).to(dtype).requires_grad_(True)
    x, ys, w = n(T, H), n(T * k, H), n(T, k)
    xs, y = tt.expert_dispatch(x, plan), tt.expert_combine(ys, w, plan)
    gs = torch.autograd.grad([xs, y], [x, ys, w], [n(T * k, H).detach(), n(T, H).detach()])
    return [xs.detach(), y.detach(), *gs]


@pytest.mark.parametrize("H,dtype", [(64, torch.bfloat16), (61, torch.bfloat16),
                                     (36, torch.float32), (33, torch.float32)])
@pytest.mark.parametrize("k", [1, 3, 4, 8])
def test_slots_outside_the_rows_are_dropped(H, dtype, k):
    T, E = 50, 6
    ids = torch.randint(0, E, (T, k), generator=torch.Generator().manual_seed(k))
    bad = torch.zeros(T, k, dtype=torch.bool)
    bad[::3, 0] = True
    bad[7] = True
    plan = tt.expert_plan(ids.to(DEV), E)
    outside = torch.tensor([T * k, T * k + 1, INT_MAX, -2, INT_MIN, 1 << 30], dtype=torch.int32)
    slots, dropped = plan.slots.clone(), plan.slots.clone()
    slots[bad.to(DEV)] = outside.repeat(T * k)[:int(bad.sum())].to(DEV)
    dropped[bad.to(DEV)] = -1
    make = lambda s: tt.ExpertPlan(s, plan.entries, plan.offsets, T, k, E)
    # rows that no slot names are not written: only those that are, are compared
    named = dropped[dropped >= 0].long()
    for i, (a, b) in enumerate(zip(everything(make(slots), T, k, H, dtype),
                                   everything(make(dropped), T, k, H, dtype))):
        assert torch.equal(a[named], b[named]) if i in (0, 3) else torch.equal(a, b)


@pytest.mark.parametrize("kept", [INT_MIN, -1, 0, 100, 101, INT_MAX])
def test_any_number_of_kept_rows(kept):
    T, k, E, H = 50, 2, 4, 24
    plan = tt.expert_plan(torch.zeros(T, k, dtype=torch.int64, device=DEV) - 1, E)   # all dropped
    plan.offsets[-1] = kept
    xs = everything(plan, T, k, H, torch.float32)[0]
    assert xs.shape == (T * k, H) and not xs[max(0, min(kept, T * k)):].any()


def test_strides():
    T, k, E, H = 40, 4, 5, 32
    plan = tt.expert_plan(torch.randint(0, E, (T, k), device=DEV), E)
    wide = torch.zeros(T, 2 * k, dtype=torch.int32, device=DEV)
    wide[:, ::2] = plan.slots
    off = torch.zeros(E + 1, 3, dtype=torch.int32, device=DEV)
    off[:, 1] = plan.offsets
    own = tt.ExpertPlan(wide[:, ::2], plan.entries, off[:, 1], T, k, E)
    for a, b in zip(everything(own, T, k, H, torch.bfloat16),
                    everything(plan, T, k, H, torch.bfloat16)):
        assert torch.equal(a, b)


def test_too_many_choices_and_another_device():
    slots = torch.zeros(2, 65, dtype=torch.int32, device=DEV)
    offsets = torch.zeros(3, dtype=torch.int32, device=DEV)
    x = torch.zeros(2, 8, device=DEV)
    with pytest.raises(RuntimeError):
        tt.expert_dispatch(x, tt.ExpertPlan(slots, None, offsets, 2, 65, 2))
    with pytest.raises(RuntimeError):
        tt.expert_dispatch(x, tt.ExpertPlan(slots[:, :2], None, offsets.cpu(), 2, 2, 2))
