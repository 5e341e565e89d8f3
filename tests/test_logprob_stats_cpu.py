"""The C ABI refuses a buffer of row statistics that is not on the 16-byte boundary
its kernels store and load at, before a device is touched."""
import pytest

from tree_training_b200 import _lib

P = 1 << 20            # a pointer that is never followed


@pytest.mark.parametrize("off", [4, 8, 12])
def test_alignment(off):
    lib = _lib.lib()
    assert lib.tt_token_logprobs_fwd(_lib.TT_F32, 4, 32, P, 32, P, 1, 1.0, 0, P, P, None, None,
                                     P + off, None) == _lib.TT_ERR_INVALID_ARG
    assert lib.tt_token_logprobs_bwd(_lib.TT_F32, 4, 32, P, 32, P, 1, 1.0, 0, None, P, P, None,
                                     P + off, P, None) == _lib.TT_ERR_INVALID_ARG
