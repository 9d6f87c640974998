"""The embedding with a factor, its gradient and its module on the GPU."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _ids(T, V, seed, hot=False):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-2, V + 2, (T,), generator=g)
    if hot:
        ids[torch.rand(T, generator=g) < 0.6] = V // 2
    return ids.to(DEV)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T,V,H", [(1, 5, 8), (4, 1000, 256), (999, 1024, 688), (3000, 64, 2048), (70000, 300, 64), (5, 3, 8200)])
@pytest.mark.parametrize("factor", [1.0, 16.0, 0.3, -2.5, 0.0])
def test_lookup_and_gradient(factor, T, V, H, dtype):
    """The row rounds once; a gradient's row is a sum of n terms in fp32 (n 2^-24), times the
    factor (2^-24), rounded once."""
    from femtotron_amd import embedding
    w = randn((V, H), 1).to(dtype).to(DEV).requires_grad_(True)
    ids = _ids(T, V, 2, hot=T > 100)
    dy = randn((T, H), 3).to(dtype).to(DEV)
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    y = embedding(ids, w, factor=factor, padding_idx=V // 3)
    ok = (ids >= 0) & (ids < V)
    want = torch.where(ok[:, None], w.detach().double()[ids.clamp(0, V - 1)] * torch.tensor(factor).double().to(DEV), 0.0)
    assert ((y.double() - want).abs() <= u * want.abs()).all()
    dw, = torch.autograd.grad(y, w, dy)
    used = ok & (ids != V // 3)
    exact = torch.zeros(V, H, dtype=torch.float64, device=DEV).index_add_(0, ids[used], dy[used].double())
    size = torch.zeros(V, H, dtype=torch.float64, device=DEV).index_add_(0, ids[used], dy[used].double().abs())
    n = torch.zeros(V, dtype=torch.float64, device=DEV).index_add_(0, ids[used], torch.ones(int(used.sum()), dtype=torch.float64, device=DEV))
    bound = u * (factor * exact).abs() + abs(factor) * size * (n[:, None] + 2) * f * (1 + u)
    assert ((dw.double() - factor * exact).abs() <= bound * (1 + 1e-9)).all()
    assert not dw[V // 3].any()


def test_factor_one_is_the_lookup():
    from femtotron_amd import embedding, ops
    w, ids = randn((100, 64), 5).bfloat16().to(DEV), _ids(50, 100, 6)
    assert torch.equal(embedding(ids, w), ops.embedding_fwd(ids, w))
    rows = embedding(ids.clamp(0, 99), w)
    assert torch.equal(rows, w[ids.clamp(0, 99)])


def test_modules_with_a_factor():
    from femtotron_amd import fuse_boundary_ops
    from femtotron_amd.boundary_ops import FusedEmbedding, unfuse_boundary_ops

    class Model(nn.Module):
        def __init__(self):
            super().__init__()
            self.embed_tokens = nn.Embedding(50, 64, padding_idx=3)

    m = Model().to(DEV, BF)
    w = m.embed_tokens.weight
    assert fuse_boundary_ops(m, embedding_factor=8.0) == 1
    e = m.embed_tokens
    assert isinstance(e, FusedEmbedding) and e.weight is w and e.factor == 8.0 and "factor" in repr(e)
    ids = torch.tensor([[1, 3], [49, 7]], device=DEV)
    y = e(ids)
    assert y.shape == (2, 2, 64) and torch.equal(y, w.detach()[ids] * 8)
    y.float().sum().backward()
    want = torch.zeros(50, 64, device=DEV)
    want[[1, 7, 49]] = 8.0
    assert torch.equal(w.grad.float(), want)
    cpu = FusedEmbedding(nn.Parameter(w.detach().cpu()), 3, 8.0)
    assert torch.equal(cpu(ids.cpu()), y.detach().cpu())
    with pytest.raises(ValueError, match="factor"):
        unfuse_boundary_ops(m)
    assert m.embed_tokens is e


def test_a_replayed_graph_and_another_stream():
    from femtotron_amd import ops
    w, dy, ids = randn((500, 64), 7).to(DEV), randn((300, 64), 8).to(DEV), _ids(300, 500, 9)
    work = lambda: (ops.embedding_fwd(ids, w, 3.0), ops.embedding_bwd(dy, ids, 500, None, 3.0))  # noqa: E731
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
    for i in range(3):
        ids.copy_(_ids(300, 500, 20 + i, hot=True))
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    from femtotron_amd import embedding
    from femtotron_amd._lib import FemtoHipError
    w, ids = randn((10, 64), 1).to(DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for args, kw, error in [((ids.int(), w), {}, ValueError), ((ids, w[:, :12]), {}, ValueError), ((ids, w.half()), {}, TypeError),
                            ((ids.cpu(), w), {}, ValueError), ((ids, w.cpu()), {}, ValueError),
                            ((ids, w), dict(factor=torch.tensor(2.0, requires_grad=True)), TypeError),
                            ((ids, w), dict(factor=float("inf")), FemtoHipError), ((ids, w), dict(factor=float("nan")), FemtoHipError)]:
        with pytest.raises(error):
            embedding(*args, **kw)
    wg = w.clone().requires_grad_(True)
    dy = torch.ones(3, 64, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(embedding(ids, wg, factor=2.0), wg, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert embedding(ids[:0], w, factor=2.0).shape == (0, 64)
