"""The norms after and before a block (block_norms) on the GPU against fp64.

Rounding counts: half a step is 2^-8 (bf16) or 2^-24 (fp32) of a stored value, once a
tensor.  In fp32 a row's sum runs over at most 16 terms a lane, 6 lane steps and 8 waves,
so with the mean, the root and the few products of a value it is off by less than FUZZ =
64 * 2^-24 of the magnitudes it adds up; the backward has two such sums in a row, and a
sum over rows adds (rows + 128) * 2^-24.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import blocks as ob
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FUZZ = 64 * 2.0 ** -24
DTYPES = (torch.bfloat16, torch.float32)
MODES = [(p, q, g) for p, q in ((True, True), (True, False), (False, True)) for g in (None, "channel", "token")]


def _ops():
    from femtotron_amd import ops
    return ops


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _inputs(rows, cols, dtype, post, pre, gate, seed=1):
    big = torch.exp2(torch.randint(-6, 6, (rows, 1), generator=torch.Generator().manual_seed(seed)).float())
    t = dict(x=randn((rows, cols), seed) * big, a=randn((rows, cols), seed + 1) * big.flip(0),
             w_post=1 + randn((cols,), seed + 2, 0.2) if post else None,
             w_pre=1 + randn((cols,), seed + 3, 0.2) if pre else None,
             gate=None if gate is None else randn((cols,) if gate == "channel" else (rows, cols), seed + 4),
             dh=randn((rows, cols), seed + 5), dy=randn((rows, cols), seed + 6) if pre else None)
    return {k: None if v is None else v.to(dtype).to(DEV) for k, v in t.items()}


def _near(name, got, ref, half, slack):
    got = _f64(got)
    assert got.shape == ref.shape, name
    off = np.abs(got - ref) - (half + 2.0 ** -23) * np.abs(ref) - slack
    assert (off <= 0).all(), f"{name}: {off.max():.3e} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


def _check(t, dtype, scale):
    ops = _ops()
    rows, cols = t["x"].shape
    half, f = HALF[dtype], {k: _f64(v) for k, v in t.items()}
    r1 = torch.empty(rows, device=DEV) if t["w_post"] is not None else None
    r2 = torch.empty(rows, device=DEV) if t["w_pre"] is not None else None
    h, y = ops.block_norms_fwd(t["x"], t["a"], t["w_post"], t["w_pre"], EPS, gate=t["gate"], scale=scale, rstd_post=r1,
                               rstd_pre=r2)
    rh, _ = ob.block_norms(f["x"], f["a"], f["w_post"], f["w_pre"], f["gate"], scale, EPS)
    _near("h", h, rh, half, FUZZ * (np.abs(f["x"]) + np.abs(rh - f["x"])))
    assert (y is None) == (t["w_pre"] is None)
    if y is not None:
        _, ry = ob.block_norms(f["x"], f["a"], f["w_post"], f["w_pre"], f["gate"], scale, EPS, h=_f64(h))
        _near("y", y, ry, half, FUZZ * np.abs(ry))
    got = dict(zip(("dx", "da", "dw_post", "dw_pre", "dgate"), ops.block_norms_bwd(
        t["dh"], t["dy"], h, t["a"], t["w_post"], t["w_pre"], gate=t["gate"], scale=scale, rstd_post=r1, rstd_pre=r2)))
    ref = ob.block_norms_bwd(f["dh"], f["dy"], _f64(h), f["a"], f["w_post"], f["w_pre"], f["gate"], scale, EPS)
    assert {k for k, v in got.items() if v is not None} == set(ref)
    for k, (v, mag) in ref.items():
        over_rows = (rows + 128) * 2.0 ** -24 if v.ndim == 1 else 0.0
        _near(k, got[k], v, half, (6 * FUZZ + over_rows) * mag)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post,pre,gate", MODES)
@pytest.mark.parametrize("rows,cols", [(1, 8), (5, 256), (9, 688), (3, 1000), (2, 1024), (33, 2048), (7, 4096), (2, 8192)])
def test_forward_and_backward(rows, cols, post, pre, gate, dtype):
    _check(_inputs(rows, cols, dtype, post, pre, gate), dtype, 0.37)


@pytest.mark.parametrize("gate", ["channel", "token"])
@pytest.mark.parametrize("rows,cols", [(4101, 512), (4500, 1024), (2100, 2048), (1050, 4096), (530, 8192)])
def test_more_rows_than_one_step_of_the_grid(rows, cols, gate):
    _check(_inputs(rows, cols, torch.bfloat16, True, True, gate, seed=11), torch.bfloat16, -1.5)


@pytest.mark.parametrize("gate", [None, "channel", "token"])
def test_autograd_and_slopes(gate):
    """fp32, through block_norms: its gradients against the slope of sum(gh h + gy y) in
    fp64 along a direction in every input."""
    from femtotron_amd import block_norms
    t = _inputs(6, 200, torch.float32, True, True, gate, seed=21)
    names = [k for k in ("x", "a", "w_post", "w_pre", "gate") if t[k] is not None]
    leaves = {k: t[k].clone().requires_grad_(True) for k in names}
    h, y = block_norms(leaves["x"], leaves["a"], leaves["w_post"], leaves["w_pre"], gate=leaves.get("gate"), scale=0.7, eps=EPS)
    grads = torch.autograd.grad((h, y), [leaves[k] for k in names], (t["dh"], t["dy"]))
    f, step = {k: _f64(v) for k, v in t.items()}, 1e-5
    d = {k: _f64(randn(tuple(t[k].shape), 31 + i)) for i, k in enumerate(names)}

    def value(s):
        v = {k: f[k] + s * d[k] for k in names}
        hh, yy = ob.block_norms(v["x"], v["a"], v["w_post"], v["w_pre"], v.get("gate"), 0.7, EPS)
        return (f["dh"] * hh).sum() + (f["dy"] * yy).sum()

    slope = (value(step) - value(-step)) / (2 * step)
    ref = ob.block_norms_bwd(f["dh"], f["dy"], _f64(h), f["a"], f["w_post"], f["w_pre"], f["gate"], 0.7, EPS)
    got = sum((_f64(g) * d[k]).sum() for k, g in zip(names, grads))
    lim = sum(((6 * FUZZ + 134 * 2.0 ** -24) * ref["d" + k][1] * np.abs(d[k])).sum() for k in names)
    # the difference: step^2 times a third derivative; h is stored in fp32, an error of 2^-24 h in it
    lim += step ** 2 * 1e6 + 2.0 ** -24 * 10 * sum(np.abs(ref["d" + k][1] * d[k]).sum() for k in names)
    assert abs(got - slope) <= lim


def test_autograd_takes_shapes_shared_gates_and_missing_gradients():
    from femtotron_amd import block_norms
    ops = _ops()
    x, a, dh, dy = (randn((2, 3, 64), s).bfloat16().to(DEV) for s in (41, 42, 43, 44))
    w1, w2 = (1 + randn((64,), s, 0.1).to(DEV) for s in (45, 46))
    w1, w2 = w1.bfloat16(), w2.bfloat16()
    g = randn((2, 1, 64), 47).bfloat16().to(DEV).requires_grad_(True)
    h, y = block_norms(x, a, w1, w2, gate=g.expand_as(x))
    (dg,) = torch.autograd.grad((h, y), [g], (dh, dy))
    full = g.detach().expand_as(x).contiguous().requires_grad_(True)
    h2, y2 = block_norms(x, a, w1, w2, gate=full)
    assert torch.equal(h, h2) and torch.equal(y, y2)
    (df,) = torch.autograd.grad((h2, y2), [full], (dh, dy))
    assert torch.equal(dg, df.sum(1, keepdim=True))
    c = randn((1, 1, 64), 48).bfloat16().to(DEV).requires_grad_(True)  # a channel gate with leading ones
    h, y = block_norms(x, a, w1, w2, gate=c)
    assert torch.autograd.grad(h.sum(), [c])[0].shape == (1, 1, 64)
    # y alone, h alone; an expanded gradient; a transposed input
    xl = x.clone().requires_grad_(True)
    h, y = block_norms(xl, a, w1, w2)
    (only_y,) = torch.autograd.grad(y, [xl], dy)
    h, y = block_norms(xl, a, w1, w2)
    (zero_h,) = torch.autograd.grad((h, y), [xl], (torch.zeros_like(dh), dy))
    assert torch.equal(only_y, zero_h)
    h, y = block_norms(xl, a, w1, None)
    assert y is None and torch.equal(torch.autograd.grad(h.sum(), [xl])[0], torch.ones_like(x))
    ht, _ = block_norms(x.transpose(0, 1), a.transpose(0, 1), w1, w2)
    assert torch.equal(ht, ops.block_norms_fwd(x, a, w1, w2, EPS)[0].transpose(0, 1))


def test_without_gate_scale_and_post_norm_it_is_add_rmsnorm():
    """h the same bits as add_rmsnorm_fwd; y off by the rounding of the normalised value that it does not make."""
    ops = _ops()
    x, a = (randn((50, 688), s).bfloat16().to(DEV) for s in (51, 52))
    w = (1 + randn((688,), 53, 0.1)).bfloat16().to(DEV)
    h, y = ops.block_norms_fwd(x, a, None, w, EPS)
    h2, y2 = ops.add_rmsnorm_fwd(x, a, w, EPS)
    assert torch.equal(h, h2)
    assert (np.abs(_f64(y) - _f64(y2)) <= 3 * 2.0 ** -8 * (1 + 2.0 ** -7) * np.abs(_f64(y2))).all()


def test_zero_rows_values_that_are_not_finite_and_determinism():
    ops = _ops()
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    r = torch.empty(0, device=DEV)
    h, y = ops.block_norms_fwd(e, e, w, w, EPS, gate=w)
    assert h.shape == y.shape == (0, 64)
    got = ops.block_norms_bwd(e, e, e, e, w, w, gate=w, rstd_post=r, rstd_pre=r)
    assert got[0].shape == (0, 64) and all(torch.count_nonzero(g) == 0 for g in got[2:])
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device=DEV)
    a = torch.zeros_like(x)
    a[1, 3], x[2, 5], a[3] = float("inf"), float("nan"), 3.0e38
    a[4] = 1e-30
    h, y = ops.block_norms_fwd(x, a, w, w, EPS)
    assert torch.count_nonzero(h[0]) == 0 and torch.count_nonzero(y[0]) == 0
    assert bool(h[1].isnan().any()) and bool(h[2, 5].isnan()) and bool(h[4:].isfinite().all())
    t = _inputs(3000, 688, torch.bfloat16, True, True, "channel", seed=61)
    r1, r2 = torch.empty(3000, device=DEV), torch.empty(3000, device=DEV)
    h, y = ops.block_norms_fwd(t["x"], t["a"], t["w_post"], t["w_pre"], EPS, gate=t["gate"], rstd_post=r1, rstd_pre=r2)
    one, two = (ops.block_norms_bwd(t["dh"], t["dy"], h, t["a"], t["w_post"], t["w_pre"], gate=t["gate"], rstd_post=r1,
                                    rstd_pre=r2) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_refusals():
    from femtotron_amd import block_norms
    from femtotron_amd._lib import FemtoHipError
    ops = _ops()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="at least one"):
        block_norms(x, x)
    with pytest.raises(ValueError, match="w_pre"):
        block_norms(x, x, w, w[:32])
    with pytest.raises(ValueError, match="gate"):
        block_norms(x, x, w, gate=torch.ones(4, 1, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="one shape"):
        block_norms(x, x[:2], w)
    with pytest.raises(TypeError, match="mismatch"):
        block_norms(x, x, w.float())
    with pytest.raises(TypeError, match="float16"):
        block_norms(x.half(), x.half(), w.half())
    with pytest.raises(ValueError, match="HIP device"):
        block_norms(x.cpu(), x.cpu(), w.cpu())
    with pytest.raises(FemtoHipError, match="multiple of 8"):
        block_norms(x[:, :60].contiguous(), x[:, :60].contiguous(), w[:60])
    with pytest.raises(ValueError, match="rstd_post"):
        ops.block_norms_bwd(x, x, x, x, w, w, rstd_pre=torch.ones(4, device=DEV))
    with pytest.raises(TypeError, match="gate"):
        block_norms(x, x, w, scale=torch.ones((), device=DEV, requires_grad=True))
    with pytest.raises(ValueError, match="needs dy"):
        ops.block_norms_bwd(x, None, x, x, None, w, rstd_pre=torch.ones(4, device=DEV))


def test_another_stream_and_a_replayed_graph():
    ops = _ops()
    t = _inputs(700, 2048, torch.bfloat16, True, True, "channel", seed=71)
    r1, r2 = torch.empty(700, device=DEV), torch.empty(700, device=DEV)

    def step():
        h, y = ops.block_norms_fwd(t["x"], t["a"], t["w_post"], t["w_pre"], EPS, gate=t["gate"], scale=0.5, rstd_post=r1,
                                   rstd_pre=r2)
        return (h, y, *ops.block_norms_bwd(t["dh"], t["dy"], h, t["a"], t["w_post"], t["w_pre"], gate=t["gate"], scale=0.5,
                                           rstd_post=r1, rstd_pre=r2))

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for k in range(4):
        new = _inputs(700, 2048, torch.bfloat16, True, True, "channel", seed=80 + k)
        for n, v in new.items():
            t[n].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(p, q) for p, q in zip(kept, step())), k


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last rows equal those of a call on them alone."""
    ops = _ops()
    rows, cols = (1 << 19) + 3, 8192
    w = (1 + randn((cols,), 91, 0.1)).bfloat16().to(DEV)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-3:] = randn((3, cols), 92).bfloat16().to(DEV)
    tail = x[-3:].clone()
    r1, r2, s1, s2 = (torch.empty(n, device=DEV) for n in (rows, rows, 3, 3))
    h, y = ops.block_norms_fwd(x, x, w, w, EPS, rstd_post=r1, rstd_pre=r2)
    ht, yt = ops.block_norms_fwd(tail, tail, w, w, EPS, rstd_post=s1, rstd_pre=s2)
    assert torch.equal(h[-3:], ht) and torch.equal(y[-3:], yt) and torch.equal(r1[-3:], s1) and torch.equal(r2[-3:], s2)
    del y
    dx, da, *_ = ops.block_norms_bwd(x, x, h, x, w, w, rstd_post=r1, rstd_pre=r2)
    dxt, dat, *_ = ops.block_norms_bwd(tail, tail, ht, tail, w, w, rstd_post=s1, rstd_pre=s2)
    assert torch.equal(dx[-3:], dxt) and torch.equal(da[-3:], dat)


def test_a_second_derivative_is_refused():
    from femtotron_amd import block_norms
    x, g = (randn((4, 64), s).to(DEV).requires_grad_(True) for s in (93, 94))
    h, _ = block_norms(x, x, torch.ones(64, device=DEV))
    (dx,) = torch.autograd.grad(h, [x], g, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_a_step_with_its_backward_in_a_graph():
    """block_norms and its gradients captured together, on leaves that no eager graph holds."""
    from femtotron_amd import block_norms
    t = _inputs(300, 688, torch.bfloat16, True, True, "token", seed=101)
    names = ["x", "a", "w_post", "w_pre", "gate"]

    def step(leaves):
        h, y = block_norms(leaves["x"], leaves["a"], leaves["w_post"], leaves["w_pre"], gate=leaves["gate"], scale=0.5)
        return [h.detach(), y.detach(), *torch.autograd.grad((h, y), [leaves[n] for n in names], (t["dh"], t["dy"]))]

    def fresh():
        return {n: t[n].clone().requires_grad_(True) for n in names}

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    held = fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(held)
    for k in range(4):
        new = _inputs(300, 688, torch.bfloat16, True, True, "token", seed=110 + k)
        with torch.no_grad():
            for n, v in new.items():
                t[n].copy_(v)
            for n in names:
                held[n].copy_(t[n])
        g.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(p, q) for p, q in zip(kept, step(fresh()))), k
