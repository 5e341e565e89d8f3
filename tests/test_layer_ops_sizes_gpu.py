"""Sizes that do not fit the 32 bits of the C ABI are refused, not cut off.  (The
tensors are expanded ones of a few bytes.)"""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BIG = 1 << 32


def zeros(*shape, to, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device=DEV).expand(*to)


def test_token_logprobs():
    with pytest.raises(ValueError):
        tt.token_logprobs(zeros(1, 1, to=(1, BIG + 5)))
    with pytest.raises(ValueError):
        tt.token_logprobs(torch.zeros(1, 8, device=DEV),
                          zeros(1, 1, to=(1, BIG + 1), dtype=torch.int64))


def test_apply_rotary():
    pos, table = torch.zeros(1, dtype=torch.int64, device=DEV), tt.rotary_table(4, 8, device=DEV)
    with pytest.raises(ValueError):
        tt.apply_rotary(zeros(1, 1, 1, to=(1, 1, BIG + 64)), None, pos, table)
    with pytest.raises(ValueError):
        tt.apply_rotary(zeros(1, 1, 8, to=(1, BIG + 1, 8)), None, pos, table)
    with pytest.raises(ValueError):
        tt.apply_rotary(zeros(1, 1, 8, to=(1, 1, 8)), zeros(1, 1, 8, to=(1, BIG + 1, 8)), pos,
                        table)


def test_experts():
    plan = tt.expert_plan(torch.zeros(1, 1, dtype=torch.int64, device=DEV), 2)
    with pytest.raises(ValueError):
        tt.expert_dispatch(zeros(1, 1, to=(1, BIG + 8)), plan)
    with pytest.raises(ValueError):
        tt.expert_combine(zeros(1, 1, to=(1, BIG + 8)), torch.ones(1, 1, device=DEV), plan)
