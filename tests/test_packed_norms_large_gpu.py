"""The packed norms past 2^32 elements: the last rows equal those of calls on them alone, bit for bit
(a row's result does not depend on which step of the grid computes it)."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5


@pytest.mark.parametrize("llama", [False, True])
def test_offsets_past_32_bits(llama):
    from femtotron_amd import ops
    rows, cols, n = (1 << 19) + 5, 8192, 3
    w = (1 + randn((cols,), 1, 0.1)).bfloat16().to(DEV)
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-n:] = randn((n, cols), 2).bfloat16().to(DEV)
    tail, r, rt = x[-n:].clone(), torch.empty(rows, device=DEV), torch.empty(n, device=DEV)
    how = dict(llama_rounding=llama)
    y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, "e4m3", rstd=r, **how)
    yt, pt = ops.rmsnorm_fwd_pack8(tail, w, EPS, "e4m3", rstd=rt, **how)
    assert torch.equal(y[-n:], yt) and torch.equal(r[-n:], rt) and torch.equal(p.exps[-n:], pt.exps)
    assert torch.equal(p.codes[-n:].view(torch.uint8), pt.codes.view(torch.uint8))
    del y
    y = ops.rmsnorm_fwd8(p, w, EPS, rstd=r, **how)
    yt = ops.rmsnorm_fwd8(pt, w, EPS, rstd=rt, **how)
    assert torch.equal(y[-n:], yt) and torch.equal(r[-n:], rt) and torch.count_nonzero(y[:-n]) == 0
    del y
    h, z = ops.add_rmsnorm_fwd8(p, x, w, EPS, **how)
    ht, zt = ops.add_rmsnorm_fwd8(pt, tail, w, EPS, **how)
    assert torch.equal(h[-n:], ht) and torch.equal(z[-n:], zt)
    del h, z
    dx, _ = ops.rmsnorm_bwd8(x, p, w, EPS, rstd=r, dres=x, **how)
    dxt, _ = ops.rmsnorm_bwd8(tail, pt, w, EPS, rstd=rt, dres=tail, **how)
    assert torch.equal(dx[-n:], dxt)
