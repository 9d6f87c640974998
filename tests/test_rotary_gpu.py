"""Rotary positions on the GPU against fp64.

Rounding counts: cos and sin are off by less than 2^-27 (the polynomials) and 4 * 2^-24
(the remainder's and their own roundings, the factor); the angle of a position below 2^24
by 2^-28.  An output is a sum of two products, rounded once: half a step of it, and 8 *
2^-24 of factor (|x0| + |x1|).  Passing dims keep their bits.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import blocks as ob
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _ops():
    from femtotron_amd import ops
    return ops


def _f64(t):
    return t.detach().double().cpu().numpy()


def _freq(rot, theta=1e4):
    from femtotron_amd import rotary_frequencies
    return rotary_frequencies(rot, theta, device=DEV)[0]


def _check(got, x, pos, f, hd, off, layout, factor, back=False):
    ref, mag = ob.rotary(_f64(x), _f64(pos), _f64(f), hd, off, layout, factor, back)
    half = HALF[x.dtype]
    err = np.abs(_f64(got) - ref)
    lim = np.where(mag > 0, half * np.abs(ref) + (1 + half) * 8 * 2.0 ** -24 * mag, 0.0)
    assert got.shape == x.shape and (err <= lim).all(), float((err - lim).max())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot,off", [(64, 64, 0), (128, 64, 64), (128, 128, 0), (96, 48, 0), (80, 40, 40), (80, 80, 0),
                                        (256, 256, 0), (32, 16, 8), (10, 6, 3), (2, 2, 0), (192, 64, 128), (1024, 1024, 0)])
def test_forward_and_backward(hd, rot, off, layout, dtype):
    ops = _ops()
    T, nq, nk = 37, 5, 2
    f, pos = _freq(rot), torch.randint(0, 1 << 24, (T,), generator=torch.Generator().manual_seed(1)).to(DEV)
    pos[:3] = torch.tensor([0, 1, -5])
    q, k = randn((T, nq * hd), 2).to(dtype).to(DEV), randn((T, nk * hd), 3).to(dtype).to(DEV)
    how = dict(head_dim=hd, rot_dim=rot, offset=off, layout=layout, factor=1.25)
    for op, back in ((ops.rotary_fwd, False), (ops.rotary_bwd, True)):
        qo, ko = op(q, k, pos, f, **how)
        _check(qo, q, pos, f, hd, off, layout, 1.25, back)
        _check(ko, k, pos, f, hd, off, layout, 1.25, back)
        q2, k2 = q.clone(), k.clone()
        got = op(q2, k2, pos, f, **how, out=(q2, k2))  # in place
        assert got[0] is q2 and torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("T", [1, 2, 3, 129, 4099])
@pytest.mark.parametrize("nq,nk", [(32, 8), (1, 0), (0, 3), (71, 1), (128, 128)])
def test_tokens_heads_and_one_side_alone(T, nq, nk):
    if T > 200 and nq + nk > 80:
        T = 300
    ops = _ops()
    f, pos = _freq(32), torch.arange(T, device=DEV) * 7
    q = randn((T, nq * 32), 4).bfloat16().to(DEV) if nq else None
    k = randn((T, nk * 32), 5).bfloat16().to(DEV) if nk else None
    qo, ko = ops.rotary_fwd(q, k, pos, f, head_dim=32)
    for t, o in ((q, qo), (k, ko)):
        assert (t is None) == (o is None)
        if t is not None:
            _check(o, t, pos, f, 32, 0, "half", 1.0)


@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 8), (0, 4), (4, 12), (1, 3)])
@pytest.mark.parametrize("dtype", HALF)
def test_strides_and_alignments(shift, pad, dtype):
    """Column views of a wider buffer, aligned for accesses of 8 elements, of 4, and of one;
    what lies around them stays."""
    ops = _ops()
    T, hd = 19, 64
    W = shift + 6 * hd + pad
    f, pos = _freq(hd), torch.arange(T, device=DEV)
    buf = randn((T, W), 6).to(dtype).to(DEV)
    before = buf.clone()
    q, k = buf[:, shift:shift + 4 * hd], buf[:, shift + 4 * hd:shift + 6 * hd]
    for layout in ("half", "interleaved"):
        qo, ko = ops.rotary_fwd(q, k, pos, f, head_dim=hd, layout=layout)
        assert torch.equal(buf, before) and qo.is_contiguous()
        _check(qo, q, pos, f, hd, 0, layout, 1.0)
        _check(ko, k, pos, f, hd, 0, layout, 1.0)
        work = before.clone()
        v = work[:, shift:shift + 4 * hd], work[:, shift + 4 * hd:shift + 6 * hd]
        ops.rotary_fwd(*v, pos, f, head_dim=hd, layout=layout, out=v)
        assert torch.equal(v[0], qo) and torch.equal(v[1], ko)
        assert torch.equal(work[:, :shift], before[:, :shift]) and torch.equal(work[:, shift + 6 * hd:], before[:, shift + 6 * hd:])


def test_positions_of_equal_sequences_and_empty_calls():
    ops = _ops()
    f, q = _freq(64), randn((24, 128), 7).bfloat16().to(DEV)
    pos = torch.randint(0, 5000, (8,), generator=torch.Generator().manual_seed(2)).to(DEV)
    a, _ = ops.rotary_fwd(q, None, pos, f, head_dim=64)
    b, _ = ops.rotary_fwd(q, None, pos.repeat(3), f, head_dim=64)
    assert torch.equal(a, b)
    e, _ = ops.rotary_fwd(q[:0], None, pos[:0], f, head_dim=64)
    assert e.shape == (0, 128)


def test_it_is_the_stock_rotation_where_both_apply():
    """fp32 tables of the same angles through rope_fwd_: products of the same factors, summed
    with one rounding more each."""
    ops = _ops()
    T, hd = 200, 64
    f, pos = _freq(hd), torch.arange(T, device=DEV)
    angle = torch.cat([pos[:, None].double() * f] * 2, -1)
    q = randn((T, 4 * hd), 8).to(DEV)
    ref = ops.rope_fwd_(q.clone(), 4, hd, T, angle.cos().float(), angle.sin().float())
    got, _ = ops.rotary_fwd(q, None, pos, f, head_dim=hd)
    x = q.view(T, 4, 2, hd // 2).abs().sum(2).repeat(1, 1, 2).view(T, -1)
    assert bool(((got - ref).abs() <= 12 * 2.0 ** -24 * x).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_autograd(layout):
    """The backward is the forward's transpose: <R q, g> = <q, R^T g>; views, several leading
    dims, an expanded and a missing gradient."""
    from femtotron_amd import apply_rotary
    ops = _ops()
    B, S, hd = 2, 9, 32
    f, pos = _freq(24), torch.arange(S, device=DEV)
    how = dict(head_dim=hd, rot_dim=24, offset=4, layout=layout, factor=0.9)
    qkv = randn((B, S, 8 * hd), 9).to(DEV).requires_grad_(True)
    q, k = qkv[..., :4 * hd], qkv[..., 4 * hd:6 * hd]
    qo, ko = apply_rotary(q, k, pos, f, **how)
    assert qo.shape == q.shape and ko.shape == k.shape
    gq, gk = randn(q.shape, 10).to(DEV), randn(k.shape, 11).to(DEV)
    (g,) = torch.autograd.grad((qo, ko), [qkv], (gq, gk), retain_graph=True)
    assert torch.count_nonzero(g[..., 6 * hd:]) == 0
    ref_q, _ = ops.rotary_bwd(gq.view(B * S, -1), None, pos, f, **how)
    assert torch.equal(g[..., :4 * hd].reshape(B * S, -1), ref_q)
    left = float(((qo.double() * gq).sum() + (ko.double() * gk).sum()).detach())
    right = float(((q.double() * g[..., :4 * hd]).sum() + (k.double() * g[..., 4 * hd:6 * hd]).sum()).detach())
    terms = float(((q.double().abs() * gq.abs()).sum() + (k.double().abs() * gk.abs()).sum()).detach())
    assert abs(left - right) <= 2 * 9 * 2.0 ** -24 * 4 * terms + 1e-9
    (only_k,) = torch.autograd.grad(ko.sum(), [qkv], retain_graph=True)  # expanded, and none for q
    _, ref_k = ops.rotary_bwd(None, torch.ones(B * S, 2 * hd, device=DEV), pos, f, **how)
    assert torch.count_nonzero(only_k[..., :4 * hd]) == 0 and torch.equal(only_k[..., 4 * hd:6 * hd].reshape(B * S, -1), ref_k)
    rows = randn((1, 4 * hd), 12).to(DEV).expand(B * S, -1).view(B, S, -1)
    (shared,) = torch.autograd.grad(qo, [qkv], rows)
    (full,) = torch.autograd.grad(apply_rotary(q, None, pos, f, **how)[0], [qkv], rows.contiguous())
    assert torch.equal(shared, full)


def test_refusals():
    from femtotron_amd import apply_rotary
    ops = _ops()
    f, q = _freq(64), torch.zeros(6, 128, dtype=torch.bfloat16, device=DEV)
    pos = torch.arange(6, device=DEV)
    for args, kw, err, word in (
            ((q, q.float(), pos, f), {}, TypeError, "mismatch"), ((q.half(), None, pos, f), {}, TypeError, "float16"),
            ((q, None, pos.int(), f), {}, TypeError, "int64"), ((q, None, pos, f.float()), {}, TypeError, "float64"),
            ((q, None, pos[:4], f), {}, ValueError, "multiple"), ((q, q[:3], pos, f), {}, ValueError, r"\[6,"),
            ((q[:, :100], None, pos, f), {}, ValueError, "heads"), ((None, None, pos, f), {}, ValueError, "one of"),
            ((q, None, pos, f), dict(layout="pairs"), ValueError, "layout"),
            ((q, None, pos, f), dict(rot_dim=32), ValueError, "rot_dim"),
            ((q.t(), None, pos, f), {}, ValueError, "contiguous last dim"),
            ((q, None, pos, f), dict(out=(q[:3], None)), ValueError, "shape"),
            ((q.cpu(), None, pos, f), {}, ValueError, "HIP device")):
        with pytest.raises(err, match=word):
            ops.rotary_fwd(*args, **{"head_dim": 64, **kw})
    from femtotron_amd._lib import FemtoHipError
    with pytest.raises(FemtoHipError, match="within the head"):
        apply_rotary(q, None, pos, f, head_dim=64, offset=8)
    k = torch.zeros_like(q)
    for out in ((k, q), (k, k), (q, q)):  # another operand's, or one for both
        with pytest.raises(FemtoHipError, match="overlap"):
            ops.rotary_fwd(q, k, pos, f, head_dim=64, out=out)
    both = torch.zeros(6, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(FemtoHipError, match="overlap"):  # shifted by half a head
        ops.rotary_fwd(both[:, :128], None, pos, f, head_dim=64, out=(both[:, 32:160], None))
    ops.rotary_fwd(both[:, :128], None, pos, f, head_dim=64, out=(both[:, 128:], None))  # beside it


def test_heads_in_a_dim_of_their_own_are_refused():
    """[batch, seq, heads, head_dim] and [tokens, heads, head_dim] would give heads for tokens."""
    from femtotron_amd import apply_rotary
    f, how = _freq(32), dict(head_dim=32)
    q = torch.zeros(2, 6, 4, 32, device=DEV)
    with pytest.raises(ValueError, match="in one dim"):
        apply_rotary(q, None, torch.arange(6, device=DEV), f, **how)
    with pytest.raises(ValueError, match="neither"):
        apply_rotary(q[0], None, torch.arange(6, device=DEV), f, **how)
    with pytest.raises(ValueError, match="in one dim"):
        apply_rotary(q[0, 0, 0], None, torch.arange(1, device=DEV), f, **how)
    x = randn((2, 6, 128), 18).to(DEV)
    pos = torch.randint(0, 900, (2, 6), generator=torch.Generator().manual_seed(3)).to(DEV)
    a, _ = apply_rotary(x, None, pos, f, **how)
    b, _ = apply_rotary(x.view(12, 128), None, pos.view(-1), f, **how)
    c = torch.cat([apply_rotary(x[i:i + 1], None, pos[i], f, **how)[0] for i in range(2)])
    assert torch.equal(a.view(12, 128), b) and torch.equal(a, c)


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last rows equal those turned alone."""
    ops = _ops()
    T, hd = (1 << 20) + 5, 64
    f, pos = _freq(hd), torch.arange(T, device=DEV)
    q = torch.empty(T, 65 * hd, dtype=torch.bfloat16, device=DEV)
    q[-5:] = randn((5, 65 * hd), 15).bfloat16().to(DEV)
    ref, _ = ops.rotary_fwd(q[-5:].clone(), None, pos[-5:].clone(), f, head_dim=hd)
    got, _ = ops.rotary_fwd(q, None, pos, f, head_dim=hd)
    assert torch.equal(got[-5:], ref)
    ops.rotary_fwd(q, None, pos, f, head_dim=hd, out=(q, None))
    assert torch.equal(q[-5:], ref)


def test_a_second_derivative_is_refused():
    from femtotron_amd import apply_rotary
    q = randn((4, 64), 16).to(DEV).requires_grad_(True)
    g = randn((4, 64), 17).to(DEV).requires_grad_(True)
    o, _ = apply_rotary(q, None, torch.arange(4, device=DEV), _freq(64), head_dim=64)
    (dq,) = torch.autograd.grad(o, [q], g, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.sum().backward()


def test_another_stream_and_a_replayed_graph():
    ops = _ops()
    f, pos = _freq(64), torch.arange(300, device=DEV)
    q, k = (torch.empty(300, n * 64, dtype=torch.bfloat16, device=DEV) for n in (8, 2))

    def step():
        a, b = ops.rotary_fwd(q, k, pos, f, head_dim=64)
        return (a, b, *ops.rotary_bwd(a, b, pos, f, head_dim=64))

    q.copy_(randn(q.shape, 13)), k.copy_(randn(k.shape, 14))
    ref, side = step(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for i in range(4):
        q.copy_(randn(q.shape, 20 + i)), k.copy_(randn(k.shape, 30 + i)), pos.add_(1000 * i)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), i
