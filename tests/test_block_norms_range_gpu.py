"""block_norms where products leave fp32's range that the formula's do not: h = x + (scale gate)
((a r) w_post), r = 1 / sqrt(mean(a^2) + eps), in that order of products."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5


@pytest.mark.parametrize("gate", [None, "channel", "token"])
@pytest.mark.parametrize("rows,cols", [(3, 64), (2, 2048), (2, 8192)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_whose_squares_overflow_adds_nothing(rows, cols, gate, dtype):
    """The mean square is infinite and r is 0, so a r w is 0 whatever a w and a w gate would be."""
    from femtotron_amd import block_norms
    x = randn((rows, cols), 1).to(dtype).to(DEV)
    a = torch.full_like(x, 1.5e38)
    a[:, ::3] = -2.5e38
    w = torch.full((cols,), 4.0, dtype=dtype, device=DEV)
    g = None if gate is None else torch.full((cols,) if gate == "channel" else (rows, cols), 3.0, dtype=dtype, device=DEV)
    w_pre = (1 + randn((cols,), 2, 0.1)).to(dtype).to(DEV)
    h, y = block_norms(x, a, w, w_pre, gate=g, scale=2.0)
    assert torch.equal(h, x)
    assert torch.equal(y, block_norms(x, torch.zeros_like(a), w, w_pre, gate=g, scale=2.0)[1])


@pytest.mark.parametrize("gate", ["channel", "token"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_gate_that_the_scale_brings_back_into_range(gate, dtype):
    """Without a norm after the block: scale gate = 2 and 2 a is finite where gate a is not.  Powers of
    two and 0: exact."""
    from femtotron_amd import block_norms
    x = torch.zeros(4, 64, dtype=dtype, device=DEV)
    a = torch.full_like(x, 2.0 ** 126)
    g = torch.full((64,) if gate == "channel" else (4, 64), 8.0, dtype=dtype, device=DEV)
    h, _ = block_norms(x, a, None, torch.ones(64, dtype=dtype, device=DEV), gate=g, scale=0.25)
    assert torch.equal(h, torch.full_like(x, 2.0 ** 127))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_large_weight_on_a_small_row(dtype):
    """h r w_pre is 2^-40 * 316 * 2^125, finite, where r w_pre is not.  Half a step of the dtype and
    a few of fp32's (the mean of equal squares is exact up to 64 additions)."""
    from femtotron_amd import block_norms
    x = torch.full((3, 64), 2.0 ** -40, dtype=dtype, device=DEV)
    w = torch.full((64,), 2.0 ** 125, dtype=dtype, device=DEV)
    _, y = block_norms(x, torch.zeros_like(x), None, w)
    ref = 2.0 ** 85 / (2.0 ** -80 + EPS) ** 0.5
    assert float((y.double() / ref - 1).abs().max()) <= torch.finfo(dtype).eps / 2 + 80 * 2.0 ** -24


@pytest.mark.parametrize("gate", [None, "channel", "token"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_gradients_of_a_row_whose_squares_overflow(gate, dtype):
    """r is 0, so nothing reaches a, its weight or its gate; dx is what it is for a row of zeros in a."""
    from femtotron_amd import block_norms
    rows, cols = 3, 2048
    g = None if gate is None else torch.full((cols,) if gate == "channel" else (rows, cols), 3.0, dtype=dtype, device=DEV)
    w, w_pre = torch.full((cols,), 4.0, dtype=dtype, device=DEV), (1 + randn((cols,), 2, 0.1)).to(dtype).to(DEV)
    dh, dy = (randn((rows, cols), s).to(dtype).to(DEV) for s in (3, 4))
    grads = []
    for fill in (1.5e38, 0.0):
        x = randn((rows, cols), 1).to(dtype).to(DEV)
        t = [v.clone().requires_grad_(True) for v in (x, torch.full_like(x, fill), w, w_pre) + (() if g is None else (g,))]
        h, y = block_norms(*t[:4], gate=None if g is None else t[4], scale=2.0)
        grads.append(torch.autograd.grad((h, y), t, (dh, dy)))
    (dx, da, dw, dw_pre, *dg), (dx0, _, _, dw_pre0, *_) = grads
    assert torch.equal(dx, dx0) and torch.equal(dw_pre, dw_pre0)
    assert all(torch.count_nonzero(v) == 0 for v in (da, dw, *dg))  # a NaN counts
