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


def _compare(B, n, room, lengths, nh, nkv, hd, dtype, *, seed=0, std=1.0, window=None, **score):
    from femtotron_amd import cache_attention
    q, k, v = _inputs(B, n, room, nh, nkv, hd, dtype, seed, std)
    for b, length in enumerate(lengths):  # what lies behind a sequence is never looked at
        k[b, max(length, 0):] = float("nan")
        v[b, max(length, 0):] = float("inf")
    want, tol = _expect(q, k, v, lengths, hd, dtype, window, **score)
    got = cache_attention(q, k, v, torch.tensor(lengths, device=DEV), head_dim=hd, window=window, **score)
    mr.check(got, want, tol, "o")
    for b, length in enumerate(lengths):
        none = max(n - max(min(length, room), 0), 0)
        assert not got[b, :none].any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 32), (8, 1, 64), (4, 4, 64), (16, 2, 128), (8, 8, 128), (1, 1, 32)])
@pytest.mark.parametrize("n", [1, 2, 5, 16])
def test_heads_and_new_tokens(n, nh, nkv, hd, dtype):
    _compare(5, n, 2300, [2300, 513, 0, 40, 1], nh, nkv, hd, dtype, seed=30 + n)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("score", [dict(cap=5.0), dict(slopes=True), dict(cap=30.0, slopes=True), dict(scale=0.4), dict(window=1),
                                   dict(window=100), dict(window=2000, cap=3.0), dict(window=7, slopes=True)], ids=str)
def test_scores_and_windows(score, hd, dtype):
    score = dict(score)
    if score.pop("slopes", None):
        score["slopes"] = torch.tensor([0.5, 0.25, 0.1, 0.01], device=DEV)
    _compare(3, 4, 2500, [2500, 1455, 2], 4, 2, hd, dtype, seed=40, std=3.0, **score)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,n,room,lengths,nh,nkv,hd,score", [
    (2, 40, 2300, [2300, 100], 8, 2, 64, dict()),
    (3, 33, 2100, [30, 2100, 0], 2, 2, 32, dict(cap=10.0)),
    (2, 300, 2600, [2600, 1000], 4, 4, 128, dict(window=150)),
    (4, 20, 5000, [3, 5000, 700, 4999], 8, 1, 64, dict(window=900, cap=20.0)),
    (1, 2200, 2100, [2100], 1, 1, 32, dict(window=64)),  # more new tokens than places: the first see nothing
    (40, 6, 2100, [2100 - 53 * b % 2100 for b in range(40)], 16, 1, 128, dict()),
])
def test_more_columns_than_a_workgroup_takes(B, n, room, lengths, nh, nkv, hd, score, dtype):
    _compare(B, n, room, lengths, nh, nkv, hd, dtype, seed=50, std=2.0, **score)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_infinities_that_a_token_does_not_see(hd, dtype):
    """A later new token's NaN, and what a window has left behind, do not reach an earlier token."""
    from femtotron_amd import cache_attention
    q, k, v = _inputs(2, 3, 2500, 4, 2, hd, dtype, 60)
    lengths = torch.tensor([2450, 1300], device=DEV)
    want, tol = _expect(q, k, v, [2450, 1300], hd, dtype, 600)
    k[0, 2449], v[0, 2449] = float("nan"), float("inf")
    k[0, :1848], v[0, :1848] = float("inf"), float("nan")  # place 1848 is the first that token 0 sees
    got = cache_attention(q, k, v, lengths, head_dim=hd, window=600)
    mr.check(got[0, :2], want[0, :2], tol[0, :2], "the tokens before")
    mr.check(got[1], want[1], tol[1], "the other sequence")
    assert got[0, 2].isnan().all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_another_stream_and_a_replayed_graph(dtype):
    from femtotron_amd import cache_attention
    q, k, v = _inputs(5, 2, 3000, 8, 2, 64, dtype, 70)
    lengths = torch.tensor([3000, 100, 1, 2999, 1000], device=DEV)
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(8)], device=DEV)
    work = lambda: cache_attention(q, k, v, lengths, head_dim=64, cap=20.0, slopes=slopes)  # noqa: E731
    ref = work().clone()
    assert torch.equal(work(), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        q.copy_(randn(q.shape, 300 + i).to(dtype))
        lengths.copy_(torch.tensor([100 + i, 3000, 0, 3 * i, 2500 - i], device=DEV))
        want = work().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
