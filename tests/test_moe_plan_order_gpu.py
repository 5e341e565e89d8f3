"""The order of ``expert_plan``: entries of one expert stay in token order however
often an expert comes up within a warp's consecutive steps, and every call gives
the same."""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def patterns(n, E):
    g = torch.Generator().manual_seed(n + E)
    i = torch.arange(n)
    return {
        "two of them": torch.randint(0, min(2, E), (n,), generator=g),
        "all": torch.randint(0, E, (n,), generator=g),
        # the first lane with an expert moves from step to step
        "another lane a step": (i % 32 + i // 32 * 5) % 32 % E,
        "one lane a step": torch.where(i % 32 == i // 32 % 32, 0, E - 1),
        "dropped between": torch.where(torch.rand(n, generator=g) < 0.5, -1, i % E),
    }


@pytest.mark.parametrize("n", [33, 257, 2047, 2049, 65536, 300001])
@pytest.mark.parametrize("E", [1, 3, 64, 1024])
def test_stable_and_the_same_every_time(n, E):
    for name, flat in patterns(n, E).items():
        ids = flat.view(n, 1).to(DEV)
        key = torch.where(flat < 0, E, flat)
        order = torch.sort(key, stable=True).indices
        kept = int((key < E).sum())
        want = torch.full((n,), -1)
        want[:kept] = order[:kept]
        want = want.to(DEV)
        for _ in range(20):
            assert torch.equal(tt.expert_plan(ids, E).entries.long(), want), name
