"""Plans of the caller's own with arrays of another type or shape are refused on
the host (before the device of the tensors is looked at, so without a GPU)."""
import pytest
import torch

import tree_training_b200 as tt

T, k, E = 4, 2, 3


def calls(slots, offsets):
    plan = tt.ExpertPlan(slots, torch.zeros(T * k, dtype=torch.int32), offsets, T, k, E)
    return (lambda: tt.expert_dispatch(torch.zeros(T, 8), plan),
            lambda: tt.expert_combine(torch.zeros(T * k, 8), torch.zeros(T, k), plan))


@pytest.mark.parametrize("slots,offsets,error", [
    (torch.int64, torch.int32, TypeError), (torch.int32, torch.int64, TypeError),
    (torch.int16, torch.int32, TypeError), (torch.float32, torch.int32, TypeError),
])
def test_types(slots, offsets, error):
    for f in calls(torch.zeros(T, k, dtype=slots), torch.zeros(E + 1, dtype=offsets)):
        with pytest.raises(error):
            f()


@pytest.mark.parametrize("slots,offsets", [
    ((T * k,), (E + 1,)), ((T, k, 1), (E + 1,)), ((T, k), (E + 1, 1)), ((T, k), (1,)), ((T, k), (0,)),
])
def test_shapes(slots, offsets):
    i32 = torch.int32
    for f in calls(torch.zeros(slots, dtype=i32), torch.zeros(offsets, dtype=i32)):
        with pytest.raises(ValueError):
            f()
