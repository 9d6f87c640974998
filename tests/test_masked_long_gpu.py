"""Attention under a mask on the GPU against fp64 in rows that take every part of the kernels: blocks
in the order of their work, pairs of heads, sums in parts of heads; under each kind of mask."""
from __future__ import annotations

import pytest
import torch

from tests import masked_reference as mr
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _compare(T, spec, nh, nkv, hd, dtype, *, seed, **score):
    from femtotron_amd import attention_mask, masked_attention
    q, do = (randn((T, nh * hd), seed + i, s).to(dtype).to(DEV) for i, s in ((0, 2.0), (3, 0.1)))
    k, v = (randn((T, nkv * hd), seed + i).to(dtype).to(DEV) for i in (1, 2))
    if score.pop("slopes", None):
        score["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], device=DEV)
    see = mr.seen(*mr.ranges(1, T, **spec), T, DEV)
    i = torch.arange(T, device=DEV)
    want, tol = mr.attention(q, k, v, see, i[:, None] - i, hd, do=do, dtype=dtype, **score)
    t = {n: None if spec.get(n) is None else torch.tensor(spec[n], device=DEV) for n in ("starts", "lengths", "prefix")}
    mask = attention_mask(1, T, t["starts"], t["lengths"], prefix=t["prefix"], window=spec.get("window"),
                          causal=spec.get("causal", True), device=DEV)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = masked_attention(q, k, v, mask, head_dim=hd, **score)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o)
    for name in want:
        mr.check(got[name], want[name], tol[name], name)
    empty, unseen = ~see.any(-1), ~see.any(0)
    assert not got["o"][empty].any() and not got["dq"][empty].any()
    assert not got["dk"][unseen].any() and not got["dv"][unseen].any()


MASKS = {
    "padded": dict(starts=[300, 1000, 1001, 1700], lengths=[250, 0, 130, 333]),  # blocks of 128 rows without a document
    "both_padded": dict(starts=[0, 900, 1400], lengths=[600, 500, 100], causal=False),
    "prefix": dict(starts=[0, 800, 805, 2000], prefix=[333, 0, 600, 10 ** 6]),
    "window": dict(starts=[0, 1500], window=300),
    "window_both": dict(starts=[100, 1500], lengths=[1300, 400], window=129, causal=False),
    "both": dict(causal=False),
}
SCORES = [dict(slopes=True), dict(cap=20.0), dict(cap=20.0, slopes=True)]


@pytest.mark.parametrize("nh,nkv,hd", [(32, 4, 64), (32, 8, 32), (32, 16, 128), (3, 1, 128)])
@pytest.mark.parametrize("name", MASKS)
def test_masks(name, nh, nkv, hd):
    _compare(2100, MASKS[name], nh, nkv, hd, BF, seed=10, **SCORES[list(MASKS).index(name) % 3])


@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("name", ["causal", "prefix", "window", "both"])
def test_a_row_long_enough_for_more_parts(name, nh, nkv, hd):
    spec = {"causal": dict(starts=[0, 4150], lengths=[4140, 50]), "prefix": dict(prefix=[4200]),
            "window": dict(window=500), "both": dict(starts=[0], lengths=[4111], causal=False)}[name]
    _compare(4200, spec, nh, nkv, hd, BF, seed=20, slopes=True)


@pytest.mark.parametrize("name", MASKS)
def test_masks_in_fp32(name):
    _compare(1100, {k: [x // 2 for x in v] if isinstance(v, list) else v for k, v in MASKS[name].items()}, 4, 2, 64, FP, seed=30,
             **SCORES[list(MASKS).index(name) % 3])
