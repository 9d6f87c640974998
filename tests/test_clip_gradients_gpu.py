"""The norm of all gradients and their clipping on the GPU against fp64."""
from __future__ import annotations

import math

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _expect(grads, max_norm):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    f = min(1.0, max_norm / (norm + 1e-6))
    return norm, f


def _close(got, g, f):
    """The factor rounds once (2^-24), the product once, to the output's type."""
    want = g.double() * f
    u = torch.finfo(got.dtype).eps / 2 + (0 if f == 1.0 else 2.0 ** -23)
    tiny = torch.finfo(got.dtype).tiny
    assert ((got.double() - want).abs() <= u * want.abs() + tiny).all()


SHAPES = [[(7,)], [(1,)], [(8192,)], [(8193,), (3, 5), (8191,)], [(100, 33), (1,), (0, 4), (2048, 512), (999,)],
          [(17,)] * 300, [(5000, 2000), (1,), (12345,)]]


@pytest.mark.parametrize("max_norm", [0.5, 1e6, 0.0])
@pytest.mark.parametrize("dtype,into", [(BF, BF), (BF, FP), (FP, FP), (FP, BF)])
@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_out_of_place(shapes, dtype, into, max_norm):
    from femtotron_amd.optim import clip_gradients, gradient_norm
    grads = [randn(s, i).to(dtype).to(DEV) for i, s in enumerate(shapes)]
    kept = [g.clone() for g in grads]
    outs = [torch.full(s, 9.0, dtype=into, device=DEV) for s in shapes]
    norm = clip_gradients(grads, max_norm, out=outs)
    want, f = _expect(grads, max_norm)
    assert norm.shape == () and norm.dtype == FP
    assert abs(float(norm) - want) <= 2.0 ** -23 * want  # the fp64 root, rounded to fp32
    assert float(gradient_norm(grads)) == float(norm)
    for g, k, o in zip(grads, kept, outs):
        assert torch.equal(g, k)
        _close(o, g, f)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_in_place(dtype):
    from femtotron_amd.optim import clip_gradients
    grads = [randn(s, i).to(dtype).to(DEV) for i, s in enumerate([(300, 77), (8192 * 3 + 5,), (2,)])]
    kept = [g.clone() for g in grads]
    norm, f = _expect(kept, 2.0)
    versions = [g._version for g in grads]
    assert abs(float(clip_gradients(grads, 2.0)) - norm) <= 2.0 ** -23 * norm
    for g, k in zip(grads, kept):
        _close(g, k, f)
    assert all(g._version > v for g, v in zip(grads, versions))
    kept = [g.clone() for g in grads]
    clip_gradients(grads, 1e9)  # nothing to clip: as they are
    assert all(torch.equal(g, k) for g, k in zip(grads, kept))


def test_mixed_types_views_and_unaligned_tensors():
    from femtotron_amd.optim import clip_gradients
    base = randn((40000,), 3).to(DEV)
    grads = [base[1:8194], base[8195:9000].view(23, 35), randn((64, 32), 4).bfloat16().to(DEV).t(),
             randn((2, 3, 4, 5), 5).to(DEV).to(memory_format=torch.channels_last), randn((100,), 6).bfloat16().to(DEV)[3:]]
    kept = [g.clone() for g in grads]
    rest = base[9000:].clone()
    norm, f = _expect(kept, 3.0)
    clip_gradients(grads, 3.0)
    for g, k in zip(grads, kept):
        _close(g, k, f)
    assert torch.equal(base[9000:], rest) and float(base[8194]) == float(randn((40000,), 3)[8194])


def test_outputs_of_mixed_strides():
    """A pair of one transposed layout beside a pair whose strides differ in a dim of one alone."""
    from femtotron_amd.optim import clip_gradients
    a, b = randn((30, 20), 7).to(DEV).t(), randn((1, 50), 8).to(DEV)
    oa, ob = torch.empty(30, 20, device=DEV).t(), torch.empty(50, device=DEV).as_strided((1, 50), (77, 1))
    norm, f = _expect([a, b], 1.0)
    clip_gradients([a, b], 1.0, out=[oa, ob])
    _close(oa, a, f)
    _close(ob, b, f)


def test_as_torch_clips():
    """torch's own clipping of the same gradients: its norm is a sum in fp32 (here of 1e5 squares:
    2^-24 times their number's root, tenfold), its factor rounded in fp32."""
    from femtotron_amd.optim import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((300, 300), (10000,), (7,))]
    for i, p in enumerate(ps):
        p.grad = randn(p.shape, 20 + i).to(DEV)
    ps.append(torch.nn.Parameter(torch.zeros(3, device=DEV)))  # without a gradient
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = None if p.grad is None else p.grad.clone()
    a, b = clip_grad_norm_(ps, 1.5), torch.nn.utils.clip_grad_norm_(qs, 1.5)
    assert abs(float(a) - float(b)) <= 2e-5 * float(b)
    for p, q in zip(ps[:3], qs[:3]):
        assert torch.allclose(p.grad, q.grad, rtol=4e-5, atol=0)
    assert float(clip_grad_norm_(ps[0], 0.1)) > 0


def test_squares_that_overflow_or_vanish_in_fp32():
    from femtotron_amd.optim import gradient_norm
    for scale in (1e25, 1e-30):
        g = (randn((5000,), 30) * scale).to(DEV)
        want = float(g.double().square().sum().sqrt())
        assert abs(float(gradient_norm([g])) - want) <= 2.0 ** -23 * want


def test_norms_that_are_not_finite():
    """As torch's: a NaN norm makes all NaN, an infinite one 0 where a gradient is finite."""
    from femtotron_amd.optim import clip_gradients
    for bad, want in ((float("nan"), float("nan")), (float("inf"), 0.0)):
        a, b = randn((100,), 40).to(DEV), randn((100,), 41).bfloat16().to(DEV)
        a[7] = bad
        norm = clip_gradients([a, b], 1.0)
        assert float(norm) == bad or (bad != bad and float(norm) != float(norm))
        assert (b.isnan().all() if want != want else not b.any()) and a[7].isnan()


def test_calls_are_the_same_bits_again_and_on_another_stream():
    from femtotron_amd.optim import clip_gradients
    grads = [randn(s, 50 + i).bfloat16().to(DEV) for i, s in enumerate([(3000, 500), (77,), (90000,)])]
    outs = [[torch.empty(g.shape, device=DEV) for g in grads] for _ in range(3)]
    norms = [clip_gradients(grads, 1.0, out=o) for o in outs[:2]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norms.append(clip_gradients(grads, 1.0, out=outs[2]))
    torch.cuda.current_stream().wait_stream(side)
    assert len({float(n) for n in norms}) == 1
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*outs))


def test_a_replayed_graph():
    from femtotron_amd.optim import clip_gradients
    grads = [randn(s, 60 + i).to(DEV) for i, s in enumerate([(300, 50), (77,)] + [(9,)] * 120)]
    outs = [torch.empty_like(g) for g in grads]
    clip_gradients(grads, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(grads, 1.0, out=outs)
    for i in range(4):
        for j, g in enumerate(grads):
            g.copy_(randn(g.shape, 1000 * i + j))
        ref = [torch.empty_like(g) for g in grads]
        want = float(clip_gradients(grads, 1.0, out=ref))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == want and all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_refusals():
    from femtotron_amd._lib import FemtoHipError
    from femtotron_amd.optim import clip_gradients
    g = torch.ones(64, 8, device=DEV)
    for grads, out, error in [
            ([g, g], None, FemtoHipError),                                # twice
            ([g[:40], g[30:]], None, FemtoHipError),                      # overlapping
            ([g], [torch.ones(8, device=DEV).expand(64, 8)], ValueError),
            ([g], [torch.ones(8, 64, device=DEV)], ValueError), ([g], [], ValueError),
            ([g], [g.view(torch.bfloat16)[:, ::2]], ValueError), ([g.cpu()], None, ValueError),
            ([g.half()], None, TypeError), ([g[:, ::2]], None, ValueError),
            ([g[:32], g[32:]], [g[32:], g[:32]], FemtoHipError)]:         # one's output is another's gradient
        with pytest.raises(error):
            clip_gradients(grads, 1.0, out=out)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_gradients([g], bad)
    with pytest.raises((ValueError, RuntimeError, TypeError)):
        clip_gradients([torch.eye(4, device=DEV).to_sparse()], 1.0)
    assert torch.equal(g, torch.ones_like(g))
    assert float(clip_gradients([], 1.0)) == 0.0
    assert float(clip_gradients([g[:0]], 1.0)) == 0.0
