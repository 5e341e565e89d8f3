"""Temperatures near the ends of fp32 are refused
by the C ABI, before a device is touched."""
import pytest

from tree_training_b200 import _lib

P = 1 << 20            # a pointer that is never followed


@pytest.mark.parametrize("temp", [0.0, -1.0, float("nan"), float("inf"), 1e-39, 9.9e-21, 1.1e20,
                                  3e38])
def test_refused(temp):
    lib = _lib.lib()
    assert lib.tt_token_logprobs_fwd(_lib.TT_F32, 4, 32, P, 32, P, 1, temp, 0, P, P, None, None,
                                     None, None) == _lib.TT_ERR_INVALID_ARG
    assert lib.tt_token_logprobs_bwd(_lib.TT_F32, 4, 32, P, 32, P, 1, temp, 0, None, P, P, None, P,
                                     P, None) == _lib.TT_ERR_INVALID_ARG
