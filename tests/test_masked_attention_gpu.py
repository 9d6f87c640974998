"""Attention under a mask on the GPU against fp64: masks, layouts, lengths, scores, strides,
infinities where nothing looks, streams, captured graphs, refusals."""
from __future__ import annotations

import pytest
import torch

from tests import masked_reference as mr
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _inputs(T, nh, nkv, hd, dtype, seed=0, std=1.0):
    q, do = (randn((T, nh * hd), seed + i, s).to(dtype).to(DEV) for i, s in ((0, std), (3, 0.1)))
    k, v = (randn((T, nkv * hd), seed + i).to(dtype).to(DEV) for i in (1, 2))
    return q, k, v, do


def _t(x):
    return None if x is None else torch.tensor(x, device=DEV)


def _mask(batch, seq, spec):
    from femtotron_amd import attention_mask
    return attention_mask(batch, seq, _t(spec.get("starts")), _t(spec.get("lengths")), prefix=_t(spec.get("prefix")),
                          window=spec.get("window"), causal=spec.get("causal", True), device=DEV)


def _run(q, k, v, do, mask, hd, **score):
    from femtotron_amd import masked_attention
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = masked_attention(q, k, v, mask, head_dim=hd, **score)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _compare(batch, seq, spec, nh, nkv, hd, dtype, *, std=1.0, seed=0, **score):
    T = batch * seq
    q, k, v, do = _inputs(T, nh, nkv, hd, dtype, seed, std)
    see = mr.seen(*mr.ranges(batch, seq, **spec), T, DEV)
    i = torch.arange(T, device=DEV)
    want, tol = mr.attention(q, k, v, see, i[:, None] - i, hd, do=do, dtype=dtype, **score)
    got = _run(q, k, v, do, _mask(batch, seq, spec), hd, **score)
    for name in want:
        mr.check(got[name], want[name], tol[name], name)
    empty = ~see.any(-1)
    assert not got["o"].reshape(T, -1)[empty].any() and not got["dq"].reshape(T, -1)[empty].any()
    unseen = ~see.any(0)
    assert not got["dk"].reshape(T, -1)[unseen].any() and not got["dv"].reshape(T, -1)[unseen].any()


MASKS = {
    "row": dict(),
    "documents": dict(starts=[0, 1, 40, 41, 128, 200, 300], lengths=None),
    "padded": dict(starts=[3, 70, 150], lengths=[50, 0, 120]),
    "both": dict(starts=[0, 90, 91], causal=False),
    "both_padded": dict(starts=[10, 150], lengths=[64, 33], causal=False),
    "prefix": dict(starts=[0, 100, 101, 230], prefix=[33, 0, 1, 1000]),
    "window": dict(starts=[0, 170], window=37),
    "window_both": dict(starts=[0, 170], window=20, causal=False),
    "window_one": dict(window=1),
    "nothing": dict(starts=[0, 100], lengths=[0, 0]),
    "no_documents": dict(starts=[]),
}


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("name", MASKS)
def test_masks(name, dtype):
    spec = {k: v for k, v in MASKS[name].items() if v is not None}
    if spec.get("starts") == []:
        from femtotron_amd import attention_mask
        mask = attention_mask(1, 70, torch.empty(0, dtype=torch.int64, device=DEV))
        q, k, v, do = _inputs(70, 4, 2, 64, dtype)
        assert not any(t.any() for t in _run(q, k, v, do, mask, 64).values())
        return
    _compare(1, 333, spec, 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 32), (4, 4, 32), (8, 1, 64), (16, 8, 64), (3, 3, 64), (4, 2, 128), (16, 16, 128),
                                       (6, 2, 128), (1, 1, 128)])
def test_heads(nh, nkv, hd, dtype):
    _compare(2, 150, dict(lengths=[150, 131]), nh, nkv, hd, dtype, seed=10)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("seq", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_lengths(seq, hd, dtype):
    _compare(1, seq, {}, 2, 1, hd, dtype, seed=20)
    _compare(3, seq, dict(lengths=[seq, 0, seq // 2], causal=False), 2, 1, hd, dtype, seed=21)


SCORES = [dict(cap=5.0), dict(cap=50.0), dict(slopes=True), dict(cap=20.0, slopes=True), dict(scale=0.5), dict(scale=0.3, cap=2.0)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("score", SCORES, ids=str)
def test_scores(score, hd, dtype):
    nh = 4
    score = dict(score)
    if score.pop("slopes", None):
        score["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], device=DEV)
    _compare(1, 260, dict(starts=[0, 100, 180], prefix=[20, 0, 5]), nh, 2, hd, dtype, std=3.0, seed=30, **score)
    _compare(2, 100, dict(window=30, causal=False), nh, 4, hd, dtype, std=3.0, seed=31, **score)


def test_large_and_small_caps():
    """A cap that scores never reach is none, one far below them leaves its sign: within the bounds,
    which hold 2^-23 of the cap."""
    for cap in (4096.0, 500.0, 0.01):
        _compare(1, 130, {}, 2, 1, 64, BF, seed=35, std=2.0, cap=cap)
    for cap in (1e6, 1e-3):
        _compare(1, 130, {}, 2, 1, 64, FP, seed=36, std=2.0, cap=cap)


def test_a_long_row_in_every_kernel():
    """Several steps of every loop, documents that end inside tiles; heads enough to pair."""
    starts = [0, 700, 701, 1500, 1777]
    for nh, nkv, hd in ((16, 2, 64), (16, 8, 32), (16, 4, 128)):
        _compare(1, 2100, dict(starts=starts), nh, nkv, hd, BF, seed=40)


@pytest.mark.parametrize("nh,nkv,hd", [(32, 16, 128), (32, 8, 128), (16, 2, 64), (9, 3, 32)])
@pytest.mark.parametrize("starts", [[0], [0, 1000, 1600, 1700, 3333]])
def test_sums_in_parts_of_heads_by_what_the_mask_holds(starts, nh, nkv, hd):
    """Enough keys that a kv head's sums come in more parts of its heads where a row is long."""
    _compare(1, 4160, dict(starts=starts), nh, nkv, hd, BF, seed=41, cap=30.0)


def test_the_gradient_by_differences():
    """fp32, against differences of the loss in fp32 inputs and fp64 sums: the second-order term
    of a step h = 2^-7 is h^2 times third derivatives of order 1, 2^-14 of a gradient's size;
    o's own error over h is 2^-24 * 64 / 2^-7 of the sizes that are summed."""
    from femtotron_amd import masked_attention
    T, nh, nkv, hd = 20, 2, 1, 32
    q, k, v, do = _inputs(T, nh, nkv, hd, FP, 50)
    mask = _mask(1, T, dict(starts=[0, 9], prefix=[4, 0]))
    score = dict(cap=4.0, slopes=torch.tensor([0.25, 0.05], device=DEV))
    got = _run(q, k, v, do, mask, hd, **score)

    def loss(**at):
        t = dict(q=q, k=k, v=v)
        t.update(at)
        return (masked_attention(t["q"], t["k"], t["v"], mask, head_dim=hd, **score).double() * do.double()).sum()

    h = 2.0 ** -7
    for name, t in (("q", q), ("k", k), ("v", v)):
        grad = got["d" + name].double()
        for i, j in ((0, 0), (5, 7), (9, 31), (19, t.shape[1] - 1), (12, 3)):
            up, down = t.clone(), t.clone()
            up[i, j] += h
            down[i, j] -= h
            step = float(up[i, j].double() - down[i, j].double())
            diff = (loss(**{name: up}) - loss(**{name: down})) / step
            assert abs(float(diff - grad[i, j])) <= 2.0 ** -10 * float(grad.abs().max()) + 2.0 ** -10 * float(do.abs().max()), (name, i, j)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_infinities_and_nan_that_nothing_sees(hd, dtype):
    """In padding, in another document, later in the own one: each token's outputs and gradients
    are those of the tokens it sees alone."""
    T, nh, nkv = 150, 2, 1
    starts, lengths = [0, 37, 100], [37, 50, 40]
    q, k, v, do = _inputs(T, nh, nkv, hd, dtype, 60)
    clean = _run(q, k, v, do, _mask(1, T, dict(starts=starts, lengths=lengths)), hd)
    bad = [float("nan"), float("inf"), -float("inf")]
    for t, seed in ((q, 0), (k, 1), (v, 2), (do, 3)):
        t[90:100] = bad[seed % 3]     # of no document
        t[140:] = bad[(seed + 1) % 3]
    v[60, 5], v[61, 6] = bad[0], bad[1]   # in the second document: seen by its tokens from 60 on
    k[70] = bad[0]
    got = _run(q, k, v, do, _mask(1, T, dict(starts=starts, lengths=lengths)), hd)
    first, third = slice(0, 37), slice(100, 140)
    for name in clean:
        for part in (first, third):
            a, b = got[name][part].double(), clean[name][part].double()
            assert torch.isfinite(a).all(), name
            # the same values; sums that meet a masked one are taken in another order
            assert float((a - b).abs().max()) <= torch.finfo(dtype).eps * 4 * float(b.abs().max()), name
        pad = torch.cat([got[name][87:100], got[name][140:]])
        assert not pad.any(), name
    o = got["o"]
    assert torch.isfinite(o[37:60]).all() and float((o[37:60].double() - clean["o"][37:60].double()).abs().max()) \
        <= torch.finfo(dtype).eps * 4 * float(clean["o"].abs().max())
    assert o[60:70, 5].isnan().all() and (o[61:70, 6] == float("inf")).all() and torch.isfinite(o[61:70, 7:hd]).all()
    assert o[70:87].isnan().all()
    assert torch.isfinite(got["dv"][71:87]).logical_not().all()  # their weights are NaN
    dq = got["dq"]
    assert torch.isfinite(dq[37:60]).all()


def test_columns_of_a_packed_projection_and_other_layouts():
    """Views in place, transposed and unaligned tensors through copies: the same bits."""
    from femtotron_amd import masked_attention
    B, S, nh, nkv, hd = 2, 70, 4, 2, 64
    wq, wk = nh * hd, nkv * hd
    qkv = randn((B, S, wq + 2 * wk), 70).bfloat16().to(DEV)
    q, k, v = qkv.split([wq, wk, wk], -1)
    mask = _mask(B, S, dict(lengths=[70, 33]))
    ref = masked_attention(q.contiguous(), k.contiguous(), v.contiguous(), mask, head_dim=hd)
    assert torch.equal(masked_attention(q, k, v, mask, head_dim=hd), ref)
    assert torch.equal(masked_attention(q.reshape(B * S, wq), k.reshape(B * S, wk), v.reshape(B * S, wk), mask, head_dim=hd),
                       ref.view(B * S, wq))
    odd = torch.empty(B * S * wq + 1, dtype=BF, device=DEV)[1:].view(B, S, wq).copy_(q)
    turned = k.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(masked_attention(odd, turned, v, mask, head_dim=hd), ref)
    # gradients that are expanded, transposed or missing reach the backward as they are
    q, k, v = (t.detach().clone().requires_grad_(True) for t in (q, k, v))
    o = masked_attention(q, k, v, mask, head_dim=hd)
    a = torch.autograd.grad(o.sum(), (q, k, v), retain_graph=True)
    b = torch.autograd.grad(o, (q, k, v), torch.ones_like(o), retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    g = randn((S, B, wq), 71).bfloat16().to(DEV)
    a = torch.autograd.grad(o.transpose(0, 1), (q, k, v), g, retain_graph=True)
    b = torch.autograd.grad(o, (q, k, v), g.transpose(0, 1).contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_calls_are_the_same_bits_again():
    q, k, v, do = _inputs(900, 16, 2, 64, BF, 80)
    mask = _mask(1, 900, dict(starts=[0, 333, 600]))
    a, b = (_run(q, k, v, do, mask, 64, cap=30.0) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_another_stream_and_a_replayed_graph():
    from femtotron_amd import attention_mask, masked_attention, ops
    T, nh, nkv, hd = 300, 4, 2, 64
    q, k, v, do = _inputs(T, nh, nkv, hd, BF, 90)
    starts, lengths = torch.tensor([0, 120, 222], device=DEV), torch.tensor([100, 102, 78], device=DEV)
    how = dict(head_dim=hd, scale=hd ** -0.5, cap=20.0)

    def work():
        mask = attention_mask(1, T, starts, lengths)
        o, lse, low = ops.masked_attn_fwd(q, k, v, mask.table, **how)
        return (masked_attention(q, k, v, mask, head_dim=hd, cap=20.0), o, *ops.masked_attn_bwd(q, k, v, o, do, lse, low, mask.table, **how))

    ref = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        fresh = _inputs(T, nh, nkv, hd, BF, 200 + 10 * i)
        for t, f in zip((q, k, v, do), fresh):
            t.copy_(f)
        starts.copy_(torch.tensor([0, 100 + i, 200 + i], device=DEV))
        lengths.copy_(torch.tensor([90, 100, 100 - i], device=DEV))
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_documents_that_no_values_describe_stay_within_the_rows():
    """Starts that do not ascend, lengths and prefixes past everything: some mask, the call's own
    rows, finite outputs."""
    T = 200
    q, k, v, do = _inputs(T, 2, 1, 64, BF, 100)
    big = 2 ** 62
    for spec in (dict(starts=[50, 10, 300, -5], lengths=[big, -big, 7, big]), dict(starts=[-big, 100, big]),
                 dict(starts=[0, 0, 0], prefix=[big, -big, 3]), dict(lengths=[big], window=2 ** 40)):
        got = _run(q, k, v, do, _mask(1, T, spec), 64)
        torch.cuda.synchronize()
        assert all(torch.isfinite(t).all() for t in got.values())


def test_more_rows_and_columns_than_32_bits_of_bytes():
    """Row offsets past 2^31 elements: the last rows of a [T, ld] view are read and written in place."""
    from femtotron_amd import masked_attention
    T, hd, ld = 2100, 64, (1 << 20)  # 2.2e9 elements, 4.4 GB
    wide = torch.empty(T, ld, dtype=BF, device=DEV)
    x = randn((3, T, hd), 110).bfloat16().to(DEV)
    for i in range(3):
        wide[:, i * hd:(i + 1) * hd] = x[i]
    mask = _mask(1, T, dict(starts=[0, 1500]))
    a = masked_attention(wide[:, :hd], wide[:, hd:2 * hd], wide[:, 2 * hd:3 * hd], mask, head_dim=hd)
    assert torch.equal(a, masked_attention(x[0], x[1], x[2], mask, head_dim=hd))


def test_refusals():
    from femtotron_amd import attention_mask, masked_attention
    q, k, v, _ = _inputs(64, 4, 2, 64, BF)
    mask = attention_mask(1, 64, device=DEV)
    call = lambda *a, **kw: masked_attention(*a, **{"head_dim": 64, **kw})  # noqa: E731
    for args, kw, error in [
            ((q[:32], k, v, mask), {}, ValueError), ((q, k[:, :64], v, mask), {}, ValueError),
            ((q.float(), k, v, mask), {}, TypeError), ((q.half(), k.half(), v.half(), mask), {}, TypeError),
            ((q.cpu(), k.cpu(), v.cpu(), mask), {}, ValueError), ((q, k, v, mask), dict(head_dim=48), ValueError),
            ((q, k, v, mask), dict(scale=-1.0), ValueError), ((q, k, v, mask), dict(cap=0.0), ValueError),
            ((q, k, v, mask), dict(cap=float("inf")), ValueError), ((q, k, v, mask), dict(slopes=torch.ones(3, device=DEV)), ValueError),
            ((q, k, v, mask), dict(slopes=torch.ones(4)), ValueError),
            ((q, k, v, mask), dict(slopes=torch.ones(4, device=DEV, requires_grad=True)), TypeError),
            ((q, k, v, attention_mask(1, 65, device=DEV)), {}, ValueError)]:
        with pytest.raises(error):
            call(*args, **kw)
    with pytest.raises(ValueError, match="head_dim"):
        call(q, k, v, mask, head_dim=16)
    qg = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(call(qg, k, v, mask).float().square().sum(), qg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    i = torch.zeros(1, dtype=torch.int64, device=DEV)
    for args, kw, error in [
            ((1, 64, i.int()), {}, TypeError), ((1, 64, i.cpu()), {}, ValueError), ((1, 64, i, i[:0]), {}, ValueError),
            ((1, 64), dict(window=0, device=DEV), ValueError), ((1, 64, i), dict(prefix=i, causal=False), ValueError),
            ((1, 64, i), dict(prefix=i, window=3), ValueError), ((-1, 64), dict(device=DEV), ValueError),
            ((1, 64), dict(device="cpu"), ValueError), ((2, 64), dict(lengths=i, device=DEV), ValueError)]:
        with pytest.raises(error):
            attention_mask(*args, **kw)


def test_no_tokens():
    from femtotron_amd import attention_mask, masked_attention
    for batch, seq in ((0, 5), (3, 0)):
        x = torch.empty(batch, seq, 128, dtype=BF, device=DEV, requires_grad=True)
        o = masked_attention(x, x, x, attention_mask(batch, seq, device=DEV), head_dim=64)
        assert o.shape == x.shape
        o.sum().backward()
        assert x.grad.shape == x.shape
