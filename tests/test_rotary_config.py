"""rotary_frequencies on the dict of a Hugging Face config alone."""
from __future__ import annotations

import pytest
import torch

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("theta", [5e5, 1e4, 2500.0])
@pytest.mark.parametrize("scaling", [None, LLAMA3, {"rope_type": "linear", "factor": 4.0},
                                     {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096}])
def test_theta_is_the_configs(scaling, theta):
    """transformers keeps rope_theta in the dict.  HF computes the frequencies in fp32: 2^-24 * (13.2
    + 40) relative, as where theta is given beside it."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

    from femtotron_amd import rotary_frequencies
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=32768, rope_theta=theta,
                      rope_scaling=None if scaling is None else dict(scaling))
    ref = (LlamaRotaryEmbedding(cfg).inv_freq if scaling is None
           else ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")[0])
    got, _ = rotary_frequencies(128, scaling=cfg.rope_scaling)
    assert float((got / ref.double() - 1).abs().max()) <= 2.0 ** -24 * (13.2 + 40)
    both, _ = rotary_frequencies(128, theta, cfg.rope_scaling)
    assert torch.equal(both, got)


def test_two_thetas_are_refused_and_none_is_ten_thousand():
    from femtotron_amd import rotary_frequencies
    with pytest.raises(ValueError, match="rope_theta"):
        rotary_frequencies(64, 1e4, {"rope_type": "default", "rope_theta": 5e5})
    with pytest.raises(ValueError, match="theta"):
        rotary_frequencies(64, scaling={"rope_theta": 0.5})
    assert torch.equal(rotary_frequencies(64)[0], rotary_frequencies(64, 1e4)[0])
    assert torch.equal(rotary_frequencies(64, scaling={"rope_theta": None})[0], rotary_frequencies(64, 1e4)[0])
