"""How far a value kept in 8 bits is from what was packed, over the whole range of bf16 and fp32
magnitudes and of ratios within a block: the bounds that the front end documents."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import blocks as ob
from tests.conftest import ROOT  # noqa: F401  (the repository on the path)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_documented_bounds(fmt, dtype):
    rng = np.random.default_rng(9)
    top = rng.uniform(-149, 127.99, (4000, 1))  # log2 of a block's scale
    x = np.exp2(top - rng.uniform(0, 40, (4000, 32))) * rng.choice([-1.0, 1.0], (4000, 32))
    x[:, 7:8] = np.exp2(top)
    x[::5, 3] = 0.0
    x = torch.from_numpy(x).to(dtype).double().numpy()
    err = np.abs(ob.unpack8(*ob.pack8(x, fmt)) - x)
    m = np.abs(x).max(-1, keepdims=True)
    if fmt == "int8":
        lim = np.maximum(2.0 ** -7 * m, 2.0 ** -119)
    else:
        lim = np.maximum(np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -17 * m), 2.0 ** -128)
    assert np.isfinite(err).all() and (err <= lim).all(), float((err / lim).max())
