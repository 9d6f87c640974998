"""e4m3 storage of the largest finite values, without a GPU: they stay finite."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import blocks as ob
from tests.conftest import ROOT  # noqa: F401  (the repository on the path)


def top_blocks(dtype: torch.dtype) -> torch.Tensor:
    """Blocks whose largest magnitude lies in the last binade: at the border of 240 2^120 and 256
    2^120 = 2^128 on both sides, the largest finite values, small ones beside them, a short last block."""
    x = torch.zeros(7, 72, dtype=torch.float64)
    big = float(torch.finfo(dtype).max)
    x[0, :] = big
    x[1, ::2], x[1, 1::2] = -big, 1.0
    x[2, 0], x[2, 1:32] = 3.3e38, torch.linspace(2.0 ** 127, 2.0 ** 128 - 2.0 ** 120, 31).double()
    x[3, 5], x[3, 40], x[3, 71] = 248 * 2.0 ** 120, 247 * 2.0 ** 120, -249 * 2.0 ** 120
    x[4, 0], x[4, 1:32] = 225 * 2.0 ** 120, torch.logspace(-30, 38, 31).double()  # just over 448 * 2^119
    x[5, 0] = 224 * 2.0 ** 120  # the largest with the exponent below
    x[6, 64] = -big  # in the short block
    return x.clamp(-big, big).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finite_values_are_kept_finite_and_near(dtype):
    x = top_blocks(dtype).double().numpy()
    codes, exps = ob.pack8(x, "e4m3")
    back = ob.unpack8(codes, exps)
    assert exps.max() == 247
    E = np.repeat(exps.astype(int) - 127, 32, 1)[:, :72]
    assert (np.abs(back - x) <= np.maximum(2.0 ** -4 * np.abs(x), np.ldexp(1.0, E - 10))).all()
    for t in (torch.bfloat16, torch.float32):
        held = torch.from_numpy(back).to(t)
        assert bool(held.isfinite().all()) and (held.double().numpy() == back).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [7, 700])
def test_the_kernels_keep_them_so(rows, dtype):
    from femtotron_amd import ops
    x = top_blocks(dtype).repeat(rows // 7, 1)
    codes, exps = ob.pack8(x.double().numpy(), "e4m3")
    w = torch.ones(72, dtype=dtype, device="cuda:0")
    for p in (ops.pack8(x.to("cuda:0"), "e4m3"), ops.rmsnorm_fwd_pack8(x.to("cuda:0"), w, 1e-5, "e4m3")[1]):
        assert np.array_equal(p.exps.cpu().numpy(), exps)
        assert np.array_equal(p.codes.float().cpu().numpy(), codes)
        for t in (torch.bfloat16, torch.float32):
            got = ops.unpack8(p, t)
            assert bool(got.isfinite().all()) and np.array_equal(got.double().cpu().numpy(), ob.unpack8(codes, exps))
