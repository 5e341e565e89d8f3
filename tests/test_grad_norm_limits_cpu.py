"""Sizes of tensors that a launch's table could not count are refused before anything is
launched (a table without room for one tensor would be filled again and again).
"""
import pytest

from tests.test_train_ops_abi_cpu import BF16, F32, INVALID, WORKSPACE, arrays, clip, norm


@pytest.mark.parametrize("call", [norm, clip])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sizes(call, dtype):
    for size in ((1 << 43) + 1, (1 << 44) - 8191, (1 << 44) - 1, 1 << 44, (1 << 63) - 1):
        assert call(tables=arrays(n=1, dtype=dtype, size=size), n=1) == INVALID
    # (the largest goes on to the next check)
    assert call(tables=arrays(n=1, dtype=dtype, size=1 << 43), n=1, ws=None) == WORKSPACE
