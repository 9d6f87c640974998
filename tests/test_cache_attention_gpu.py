"""Attention of new tokens over a cache on the GPU against fp64."""
from __future__ import annotations

import pytest
import torch

from tests import masked_reference as mr
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _inputs(B, n, room, nh, nkv, hd, dtype, seed=0, std=1.0):
    q = randn((B, n, nh * hd), seed, std).to(dtype).to(DEV)
    k, v = (randn((B, room, nkv * hd), seed + 1 + i).to(dtype).to(DEV) for i in range(2))
    return q, k, v


def _expect(q, k, v, lengths, hd, dtype, window=None, **score):
    outs, tols = [], []
    for b, n_b in enumerate(lengths):
        n = q.shape[1]
        end = min(max(n_b, 0), k.shape[1])
        at = torch.arange(end - n, end, device=DEV)
        j = torch.arange(max(end, 1), device=DEV)
        away = at[:, None] - j
        see = (away >= 0) & (j < end)
        if window is not None:
            see &= away < window
        kb, vb = (t[b, :end] if end else torch.zeros_like(t[b, :1]) for t in (k, v))  # of no place: one that none sees
        want, tol = mr.attention(q[b], kb, vb, see, away, hd, dtype=dtype, **score)
        outs.append(want["o"])
        tols.append(tol["o"])
    return torch.stack(outs), torch.stack(tols)


def _compare(B, n, room, lengths, nh, nkv, hd, dtype, *, seed=0, std=1.0, window=None, **score):
    from femtotron_amd import cache_attention
    q, k, v = _inputs(B, n, room, nh, nkv, hd, dtype, seed, std)
    for b, length in enumerate(lengths):  # what lies behind a sequence is never looked at
        k[b, max(length, 0):] = float("nan")
        v[b, max(length, 0):] = float("inf")
    want, tol = _expect(q, k, v, lengths, hd, dtype, window, **score)
    got = cache_attention(q, k, v, torch.tensor(lengths, device=DEV), head_dim=hd, window=window, **score)
    assert got.shape == q.shape and got.dtype == dtype
    mr.check(got, want, tol, "o")
    for b, length in enumerate(lengths):
        none = max(n - max(min(length, room), 0), 0)
        assert not got[b, :none].any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 32), (8, 1, 64), (4, 4, 64), (16, 2, 128), (8, 8, 128), (1, 1, 32)])
@pytest.mark.parametrize("n", [1, 2, 5, 16])
def test_heads_and_new_tokens(n, nh, nkv, hd, dtype):
    _compare(3, n, 700, [700, 513, 40], nh, nkv, hd, dtype, seed=n)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("room", [1, 31, 32, 33, 127, 128, 129, 1000, 5000])
def test_rooms_and_lengths(room, dtype):
    lengths = [room, 0, 1, room // 2, max(room - 1, 0), room // 3]
    _compare(6, 1, room, lengths, 4, 2, 64, dtype, seed=100)
    _compare(6, 3, room, lengths, 4, 2, 64, dtype, seed=101)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("score", [dict(cap=5.0), dict(slopes=True), dict(cap=30.0, slopes=True), dict(scale=0.4),
                                   dict(window=1), dict(window=100), dict(window=1000, cap=3.0), dict(window=7, slopes=True)], ids=str)
def test_scores_and_windows(score, hd, dtype):
    score = dict(score)
    if score.pop("slopes", None):
        score["slopes"] = torch.tensor([0.5, 0.25, 0.1, 0.01], device=DEV)
    _compare(3, 4, 900, [900, 455, 2], 4, 2, hd, dtype, seed=110, std=3.0, **score)


def test_one_long_sequence_among_short_ones():
    _compare(70, 1, 6000, [6000 if b == 33 else 3 + b for b in range(70)], 8, 2, 64, BF, seed=120)


def test_more_columns_than_a_workgroup_takes():
    _compare(2, 40, 300, [300, 100], 8, 2, 64, BF, seed=130)
    _compare(2, 33, 300, [300, 30], 2, 2, 32, FP, seed=131)
    _compare(300, 20, 200, [200 - b % 190 for b in range(300)], 8, 4, 32, BF, seed=132)  # a chunk a sequence


def test_sequences_enough_for_the_chip():
    """A workgroup a sequence and head, whatever the room."""
    _compare(1100, 1, 2300, [2300 if b % 100 == 0 else 1 + 7 * b % 60 for b in range(1100)], 4, 4, 32, BF, seed=135)


def test_lengths_past_the_room_and_below_nothing():
    from femtotron_amd import cache_attention
    q, k, v = _inputs(4, 2, 300, 4, 2, 64, BF, 140)
    lengths = [2 ** 60, -7, 301, -2 ** 60]
    got = cache_attention(q, k, v, torch.tensor(lengths, device=DEV), head_dim=64)
    want, tol = _expect(q, k, v, [300, 0, 300, 0], 64, BF)
    mr.check(got, want, tol, "o")
    assert not got[1].any() and not got[3].any()


def test_layouts_of_the_cache():
    """[batch, kv heads, room, head_dim] transposed, rows of a longer cache, heads apart: the same bits."""
    from femtotron_amd import cache_attention
    B, room, nkv, hd = 2, 400, 2, 64
    q, k, v = _inputs(B, 1, room, 8, nkv, hd, BF, 150)
    lengths = torch.tensor([400, 211], device=DEV)
    ref = cache_attention(q, k, v, lengths, head_dim=hd)
    k4, v4 = (t.view(B, room, nkv, hd) for t in (k, v))
    assert torch.equal(cache_attention(q, k4, v4, lengths, head_dim=hd), ref)
    kh, vh = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k4, v4))
    assert torch.equal(cache_attention(q, kh, vh, lengths, head_dim=hd), ref)
    both = torch.cat([k, v], -1)  # keys and values in one row
    assert torch.equal(cache_attention(q, both[..., :nkv * hd], both[..., nkv * hd:], lengths, head_dim=hd), ref)
    wide = torch.zeros(B, 900, nkv * hd, dtype=BF, device=DEV)
    wide[:, :room] = k
    assert torch.equal(cache_attention(q, wide[:, :room], v, lengths, head_dim=hd), ref)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_infinities_that_a_token_does_not_see(dtype):
    """A later new token's NaN, and what a window has left behind, do not reach an earlier token."""
    from femtotron_amd import cache_attention
    q, k, v = _inputs(1, 3, 500, 4, 2, 64, dtype, 160)
    lengths = torch.tensor([450], device=DEV)
    clean = cache_attention(q, k, v, lengths, head_dim=64, window=60)
    k[0, 449], v[0, 449] = float("nan"), float("inf")
    k[0, :388], v[0, :388] = float("inf"), float("nan")  # place 388 is the first that token 0 sees
    got = cache_attention(q, k, v, lengths, head_dim=64, window=60)
    bound = torch.finfo(dtype).eps * 4 * float(clean.abs().max())
    assert float((got[0, :2].double() - clean[0, :2].double()).abs().max()) <= bound
    assert got[0, 2].isnan().all()


def test_an_answer_of_single_tokens_is_the_whole_sequence():
    """Token by token over the growing cache, as the rows of one causal call: within both bounds."""
    from femtotron_amd import attention_mask, cache_attention, masked_attention
    T, nh, nkv, hd = 70, 4, 2, 64
    q, k, v = _inputs(1, T, T, nh, nkv, hd, BF, 170)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.01], device=DEV)
    whole = masked_attention(q, k, v, attention_mask(1, T, device=DEV), head_dim=hd, cap=10.0, slopes=slopes)
    want, tol = _expect(q, k, v, [T], hd, BF, cap=10.0, slopes=slopes)
    mr.check(whole, want, tol, "whole")
    for t in range(T):
        one = cache_attention(q[:, t:t + 1], k, v, torch.tensor([t + 1], device=DEV), head_dim=hd, cap=10.0, slopes=slopes)
        mr.check(one, want[:, t:t + 1], tol[:, t:t + 1], f"token {t}")
    some = cache_attention(q[:, 50:], k, v, torch.tensor([T], device=DEV), head_dim=hd, cap=10.0, slopes=slopes)
    mr.check(some, want[:, 50:], tol[:, 50:], "the last 20")


def test_a_cache_past_2_to_the_31_elements():
    from femtotron_amd import cache_attention
    B, room, nkv, hd = 1, 300000, 64, 128  # 2.46e9 elements, 4.9 GB each
    k = torch.zeros(B, room, nkv * hd, dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    last = 700
    tk, tv = (randn((1, last, nkv * hd), 180 + i).bfloat16().to(DEV) for i in range(2))
    k[:, -last:], v[:, -last:] = tk, tv
    q = randn((B, 1, nkv * hd), 182).bfloat16().to(DEV)
    got = cache_attention(q, k, v, torch.tensor([room], device=DEV), head_dim=hd, window=last)
    assert torch.isfinite(got).all()
    want, tol = _expect(q, tk, tv, [last], hd, BF)
    mr.check(got, want, tol, "o")


def test_another_stream_and_a_replayed_graph():
    from femtotron_amd import cache_attention
    q, k, v = _inputs(5, 1, 2000, 8, 2, 64, BF, 190)
    lengths = torch.tensor([2000, 100, 1, 1999, 1000], device=DEV)
    work = lambda: cache_attention(q, k, v, lengths, head_dim=64, cap=20.0)  # noqa: E731
    ref = work().clone()
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
        q.copy_(randn(q.shape, 300 + i).bfloat16())
        lengths.copy_(torch.tensor([100 + i, 2000, 0, 3 * i, 1500 - i], device=DEV))
        want = work().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_refusals():
    from femtotron_amd import cache_attention
    q, k, v = _inputs(2, 1, 64, 4, 2, 64, BF)
    n = torch.tensor([3, 4], device=DEV)
    call = lambda *a, **kw: cache_attention(*a, **{"head_dim": 64, **kw})  # noqa: E731
    for args, kw, error in [
            ((q[0], k, v, n), {}, ValueError), ((q, k[:1], v[:1], n), {}, ValueError), ((q, k, v[:, :32], n), {}, ValueError),
            ((q, k, v, n.int()), {}, ValueError), ((q, k, v, n[:1]), {}, ValueError), ((q, k, v, n.cpu()), {}, ValueError),
            ((q.float(), k, v, n), {}, TypeError), ((q, k, v, n), dict(window=0), ValueError), ((q, k, v, n), dict(cap=-1.0), ValueError),
            ((q, k, v, n), dict(scale=0.0), ValueError), ((q, k, v, n), dict(slopes=torch.ones(2, device=DEV)), ValueError),
            ((q.clone().requires_grad_(True), k, v, n), {}, TypeError),
            ((q.detach(), k.view(2, 64, 2, 64).transpose(2, 3), v.view(2, 64, 2, 64).transpose(2, 3), n), {}, ValueError)]:
        with pytest.raises(error):
            call(*args, **kw)
    with pytest.raises(ValueError, match="head_dim"):
        call(q, k, v, n, head_dim=16)
    assert call(q[:0], k[:0], v[:0], n[:0]).shape == (0, 1, 256)
    assert call(q[:, :0], k, v, n).shape == (2, 0, 256)
    assert not call(q, k[:, :0], v[:, :0], n).any()
