"""Attention over a cache where its places are dealt out in shares that a second kernel joins, on
the GPU against fp64."""
from __future__ import annotations

import pytest
import torch

from tests import masked_reference as mr
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _inputs(B, n, room, nh, nkv, hd, dtype, seed=0, std=1.0):
    """q, k, v of a call that is answered in shares: it asks for room for their sums."""
    from femtotron_amd import _lib
    code = {BF: _lib.FH_BF16, FP: _lib.FH_F32}[dtype]
    assert _lib.lib().fh_cache_attn_workspace_size(code, B, n, room, nh, nkv, hd) > 0
    q = randn((B, n, nh * hd), seed, std).to(dtype).to(DEV)
    k, v = (randn((B, room, nkv * hd), seed + 1 + i).to(dtype).to(DEV) for i in range(2))
    return q, k, v


def _expect(q, k, v, lengths, hd, dtype, window=None, **score):
    """Outputs and bounds, sequence by sequence, over the places that its tokens see."""
    outs, tols = [], []
    n, room = q.shape[1], k.shape[1]
    for b, length in enumerate(lengths):
        end = min(max(length, 0), room)
        first = max(0, end - n + 1 - window) if window else 0
        at = torch.arange(end - n, end, device=DEV)
        j = torch.arange(first, max(end, first + 1), device=DEV)
        away = at[:, None] - j
        see = (away >= 0) & (j < end)
        if window:
            see &= away < window
        kb, vb = (t[b, first:end] if end > first else torch.zeros_like(t[b, :1]) for t in (k, v))
        want, tol = mr.attention(q[b], kb, vb, see, away, hd, dtype=dtype, **score)
        outs.append(want["o"])
        tols.append(tol["o"])
    return torch.stack(outs), torch.stack(tols)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_what_a_tile_of_columns_does_not_see_of_a_share(hd, dtype):
    """256 new tokens in a window of 64: the first share lies before all that the later tiles of
    columns see, and holds what is not finite."""
    from femtotron_amd import cache_attention
    n, room, window, nh = 256, 4096, 64, 4
    q, k, v = _inputs(1, n, room, nh, nh, hd, dtype, 10)
    want, tol = _expect(q, k, v, [room], hd, dtype, window)
    first = room - n + 1 - window
    for bad_k, bad_v in ((1.0, float("inf")), (1.0, float("nan")), (float("nan"), 1.0), (float("inf"), -float("inf"))):
        k2, v2 = k.clone(), v.clone()
        k2[0, first:first + 3] *= bad_k   # seen by tokens 0 to 65 at most
        v2[0, first:first + 3] *= bad_v
        got = cache_attention(q, k2, v2, torch.tensor([room], device=DEV), head_dim=hd, window=window)
        mr.check(got[:, 66:], want[:, 66:], tol[:, 66:], f"k {bad_k}, v {bad_v}")
        assert not torch.isfinite(got[0, :64]).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_what_a_tile_of_columns_does_not_see_of_a_short_segment(dtype):
    """A share that takes the last places of one sequence and the first two of the next, which the
    second tile of columns does not see."""
    from femtotron_amd import cache_attention
    n, room, window, nh, hd = 40, 2500, 87, 4, 64
    q, k, v = _inputs(2, n, room, nh, nh, hd, dtype, 20)
    lengths = [2000, 2500]  # 126 places each
    want, tol = _expect(q, k, v, lengths, hd, dtype, window)
    first = 2500 - n + 1 - window
    v[1, first] = float("inf")  # seen by token 0 alone
    got = cache_attention(q, k, v, torch.tensor(lengths, device=DEV), head_dim=hd, window=window)
    mr.check(got[0], want[0], tol[0], "the other sequence")
    mr.check(got[1, 1:], want[1, 1:], tol[1, 1:], "the other tokens")
    assert not torch.isfinite(got[1, 0]).any()
