"""rotary_frequencies refuses a config's dict that holds one scaling for each kind of layer."""
from __future__ import annotations

import pytest
import torch


def test_a_dict_of_layer_types_is_refused():
    from femtotron_amd import rotary_frequencies
    by_layer = {"full_attention": {"rope_type": "linear", "factor": 8.0, "rope_theta": 1e6},
                "sliding_attention": {"rope_type": "default", "rope_theta": 1e4}}
    with pytest.raises(ValueError, match="full_attention"):
        rotary_frequencies(64, scaling=by_layer)
    one, _ = rotary_frequencies(64, 1e6, {"rope_type": "linear", "factor": 8.0})
    assert torch.equal(one * 8, rotary_frequencies(64, 1e6)[0])
