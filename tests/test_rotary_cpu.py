"""``rotary_table`` (CPU) against transformers' own frequency functions for
every scaling, and its refusals."""
import math

import pytest
import torch

from tree_training_b200 import rotary_table

P = 300


def _hf(scaling, dim, theta, seq_len):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim,
                      max_position_embeddings=scaling.get("original_max_position_embeddings", 64),
                      rope_parameters={**scaling, "rope_theta": theta})
    inv, amp = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, torch.device("cpu"), seq_len=seq_len)
    return inv.double(), amp


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 64},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 64,
     "mscale": 0.707, "mscale_all_dim": 1.0, "beta_fast": 16.0, "beta_slow": 2.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 64},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 64},
])
@pytest.mark.parametrize("dim", [32, 64])
def test_scaled_tables_match_transformers(scaling, dim):
    inv, amp = _hf(scaling, dim, 1e4, P)
    t = rotary_table(P, dim, 1e4, scaling).double()
    ang = torch.arange(P, dtype=torch.float64)[:, None] * inv
    # their frequencies are fp32: an angle of 300 is off by at most 300 * 2^-22
    tol = P * 2.0 ** -22 + 1e-6
    assert (t[:, :dim // 2] - ang.cos() * amp).abs().max() < tol
    assert (t[:, dim // 2:] - ang.sin() * amp).abs().max() < tol


def test_longrope_takes_the_factors_of_its_length():
    s = {"rope_type": "longrope", "short_factor": [1.0, 2.0], "long_factor": [3.0, 5.0],
         "original_max_position_embeddings": 64, "factor": 4.0}
    amp = math.sqrt(1.0 + math.log(4.0) / math.log(64))
    for n, f in ((64, (1.0, 2.0)), (65, (3.0, 5.0))):
        t = rotary_table(n, 4, 100.0, s).double()
        ang = torch.arange(n, dtype=torch.float64)[:, None] / torch.tensor(
            [f[0], 10.0 * f[1]], dtype=torch.float64)
        assert (t - torch.cat([ang.cos(), ang.sin()], 1) * amp).abs().max() < 1e-6


def test_plain_table_is_rounded_once():
    t = rotary_table(40960, 8, 1e6)
    ang = torch.arange(40960, dtype=torch.float64)[:, None] * \
        (1e6 ** -(torch.arange(0, 8, 2, dtype=torch.float64) / 8))
    assert t.dtype == torch.float32 and t.shape == (40960, 8)
    assert torch.equal(t, torch.cat([ang.cos(), ang.sin()], 1).float())


def test_refusals():
    for a in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError):
            rotary_table(*a)
    for s in ({"rope_type": "other"}, {"rope_type": "linear", "factor": 0.5},
              {"rope_type": "yarn", "factor": 2.0},
              {"rope_type": "longrope", "short_factor": [1.0], "long_factor": [1.0],
               "original_max_position_embeddings": 8}):
        with pytest.raises(ValueError):
            rotary_table(16, 8, 1e4, s)
