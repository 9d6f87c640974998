"""Attention under a mask on the GPU: infinities and NaN that a token does not see, under every kind
of score and in long rows."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _run(q, k, v, do, mask, hd, **score):
    from femtotron_amd import masked_attention
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = masked_attention(q, k, v, mask, head_dim=hd, **score)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _inputs(T, nh, nkv, hd, dtype, seed):
    q, do = (randn((T, nh * hd), seed + i, s).to(dtype).to(DEV) for i, s in ((0, 2.0), (3, 0.1)))
    k, v = (randn((T, nkv * hd), seed + i).to(dtype).to(DEV) for i in (1, 2))
    return q, k, v, do


def _unseen(T, starts, lengths, nh, nkv, hd, dtype, seed, *, bad_document, spoil, **score):
    """All outputs and gradients of the other documents with one document, and all padding, spoilt by
    `spoil`: finite, and the values without it, but for the order of sums that meet masked places
    (two roundings each way, of values up to the largest)."""
    from femtotron_amd import attention_mask
    mask = attention_mask(1, T, torch.tensor(starts, device=DEV), torch.tensor(lengths, device=DEV))
    tensors = dict(zip(("q", "k", "v", "do"), _inputs(T, nh, nkv, hd, dtype, seed)))
    clean = _run(*tensors.values(), mask, hd, **score)
    rows = torch.zeros(T, dtype=torch.bool, device=DEV)
    for s, n in zip(starts, lengths):
        rows[s:s + n] = True
    bad = ~rows
    s, n = starts[bad_document], lengths[bad_document]
    bad[s:s + n] = True
    for name, value in spoil.items():
        tensors[name][bad] = value
    got = _run(*tensors.values(), mask, hd, **score)
    for name in clean:
        a, b = got[name][~bad].double(), clean[name][~bad].double()
        assert torch.isfinite(a).all(), name
        assert float((a - b).abs().max()) <= torch.finfo(dtype).eps * 4 * float(b.abs().max()), name
        assert not got[name][~rows].any(), name


SCORES = [dict(cap=5.0), dict(slopes=True), dict(cap=20.0, slopes=True)]
SPOILT = [dict(k=NAN), dict(k=INF, v=NAN), dict(q=NAN, do=INF), dict(q=-INF, k=INF, v=-INF, do=NAN)]


def _score(score, nh):
    score = dict(score)
    if score.pop("slopes", None):
        score["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], device=DEV)
    return score


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("spoil", SPOILT, ids=str)
def test_under_a_cap_and_a_bias(spoil, score, hd, dtype):
    _unseen(150, [0, 37, 100], [37, 50, 40], 2, 1, hd, dtype, 60, bad_document=1, spoil=spoil, **_score(score, 2))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("score", SCORES, ids=str)
def test_a_later_key_of_the_own_document(score, hd, dtype):
    """A causal row's later keys, NaN, reach neither the outputs nor dq of the rows before them."""
    from femtotron_amd import attention_mask
    T, at = 100, 70
    score = _score(score, 2)
    mask = attention_mask(1, T, device=DEV)
    q, k, v, do = _inputs(T, 2, 1, hd, dtype, 80)
    clean = _run(q, k, v, do, mask, hd, **score)
    k[at:] = NAN
    got = _run(q, k, v, do, mask, hd, **score)
    for name in ("o", "dq"):
        a, b = got[name][:at].double(), clean[name][:at].double()
        assert torch.isfinite(a).all(), name
        assert float((a - b).abs().max()) <= torch.finfo(dtype).eps * 4 * float(b.abs().max()), name
        assert got[name][at:].isnan().all(), name


@pytest.mark.parametrize("nh,nkv,hd", [(32, 4, 64), (32, 8, 32), (32, 8, 128)])
@pytest.mark.parametrize("score", [dict(), dict(cap=20.0)], ids=str)
@pytest.mark.parametrize("spoil", SPOILT, ids=str)
def test_in_rows_of_every_kernel(spoil, score, nh, nkv, hd):
    """Blocks in the order of their work, pairs of heads, sums in parts of heads."""
    _unseen(2200, [0, 700, 1100, 1500], [700, 400, 370, 500], nh, nkv, hd, BF, 90, bad_document=1, spoil=spoil, **score)


@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("score", [dict(), dict(cap=20.0)], ids=str)
def test_beside_a_row_long_enough_for_more_parts(score, nh, nkv, hd):
    _unseen(4600, [0, 4200], [4200, 300], nh, nkv, hd, BF, 100, bad_document=1, spoil=dict(q=NAN, k=-INF, v=INF, do=NAN), **score)
