"""``rotary_table`` with a config's ``rope_parameters``, which name the base too."""
import pytest
import torch

from tree_training_b200 import rotary_table


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 16},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 16},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 16},
])
def test_the_base_of_the_parameters(scaling):
    own = dict(scaling, rope_theta=5e5)
    want = rotary_table(64, 32, 5e5, scaling)
    assert torch.equal(rotary_table(64, 32, scaling=own), want)
    assert torch.equal(rotary_table(64, 32, 5e5, own), want)
    # one that is given stands; without either it is 10,000
    assert torch.equal(rotary_table(64, 32, 1e4, own), rotary_table(64, 32, 1e4, scaling))
    assert torch.equal(rotary_table(64, 32, scaling=scaling), rotary_table(64, 32, 1e4, scaling))
    assert not torch.equal(want, rotary_table(64, 32, 1e4, scaling))


def test_a_config_of_transformers():
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=64, num_attention_heads=2,
                      rope_parameters={"rope_type": "linear", "factor": 4.0, "rope_theta": 5e5})
    inv = 5e5 ** -(torch.arange(0, 32, 2, dtype=torch.float64) / 32) / 4
    ang = torch.arange(64, dtype=torch.float64)[:, None] * inv
    t = rotary_table(64, 32, scaling=cfg.rope_parameters).double()
    assert (t - torch.cat([ang.cos(), ang.sin()], 1)).abs().max() < 1e-6
