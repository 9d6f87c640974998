"""The norms around a block on more rows than one step of their grids takes: the loops over rows, the
next row's loads, the sums that pass between the waves of a row, a ragged last step.

Shapes by the largest grids (blocks x rows of a step): the backward of a packed x 256 x 8, 8, 4, 2
and 1 rows at up to 512, 1024, 2048, 4096 and 8192 columns (fp32 up to 2048 columns 512 x 4); the norm
of a packed x 1024 x 4 rows at 1025 to 2048 bf16 columns, 512 x 4 at up to 4096, 512 x 2 at 8192; its
add + norm 768 x 4, and x 2 at 8192 bf16 columns; fp32 rows shared by two and four waves 512 x 2 and
512 x 1, add + norm 768 x 2 and 768 x 1.

Rounding counts as in test_packed8_gpu.py: half a step is 2^-8 (bf16) or 2^-24 (fp32); a row's sum with
its mean, root and product under 144 * 2^-24 relative; a sum over rows under (rows + 128) * 2^-24 of
its terms' magnitudes.  The reference is torch's elementary operations in fp64.
"""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn
from tests.test_block_norms_gpu import _check, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FUZZ = 144 * 2.0 ** -24
BF16, FP32 = torch.bfloat16, torch.float32


def _ops():
    from femtotron_amd import ops
    return ops


def _rows(rows, cols, seed, dtype, sizes=True):
    g = torch.Generator(DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV)
    if sizes:  # rows of many sizes, some channels far above the rest
        x *= torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g, device=DEV).float())
        x[:, ::37] *= 300
    return x.to(dtype)


def _norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def _within(name, got, ref, lim):
    over = (got.double() - ref).abs() - lim
    assert got.shape == ref.shape and bool((over <= 0).all()), f"{name}: {float(over.max()):.3e} over its bound"


@pytest.mark.parametrize("dtype,rows,cols,fmt", [
    (BF16, 2061, 512, "int8"), (BF16, 4109, 1000, "e4m3"), (BF16, 4101, 2048, "int8"), (BF16, 1030, 1096, "e4m3"),
    (BF16, 3077, 4096, "e4m3"), (BF16, 517, 4096, "int8"), (BF16, 1541, 8192, "int8"), (BF16, 1029, 5000, "e4m3"),
    (BF16, 261, 8192, "e4m3"), (FP32, 3077, 2048, "int8"), (FP32, 2061, 256, "e4m3"), (FP32, 1541, 4096, "e4m3"),
    (FP32, 1029, 2056, "int8"), (FP32, 773, 8192, "int8"), (FP32, 517, 8192, "e4m3")])
def test_packed_norms_rounded_once(dtype, rows, cols, fmt):
    ops = _ops()
    x, half = _rows(rows, cols, 1, dtype), HALF[dtype]
    a, dy, dres = (_rows(rows, cols, s, dtype, sizes=False) for s in (2, 3, 4))
    w = (1 + randn((cols,), 5, 0.1)).to(dtype).to(DEV)
    r0, r1, r2 = (torch.empty(rows, device=DEV) for _ in range(3))
    y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, fmt, rstd=r0)
    q = ops.pack8(x, fmt)
    assert torch.equal(p.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(p.exps, q.exps)
    kept, w64, tol = ops.unpack8(p, FP32).double(), w.double(), half + FUZZ
    ref = _norm(x.double(), w64)
    _within("y", y, ref, tol * ref.abs())
    root = (x.double().square().mean(-1) + EPS).rsqrt()
    _within("rstd", r0, root, FUZZ * root)
    ref = _norm(kept, w64)
    _within("y8", ops.rmsnorm_fwd8(p, w, EPS, rstd=r1), ref, tol * ref.abs())
    h, z = ops.add_rmsnorm_fwd8(p, a, w, EPS, rstd=r2)
    s = kept + a.double()
    _within("h", h, s, (half + 2.0 ** -24) * s.abs())
    ref = _norm(h.double(), w64)
    _within("z", z, ref, tol * ref.abs())
    root = (h.double().square().mean(-1) + EPS).rsqrt()
    _within("rstd of h", r2, root, FUZZ * root)
    r = (kept.square().mean(-1, keepdim=True) + EPS).rsqrt()
    g, n = dy.double() * w64, kept * r
    dx = r * (g - n * (g * n).mean(-1, keepdim=True))
    terms = r * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    over = (dy.double() * n).abs().sum(0)
    dw = (dy.double() * n).sum(0)
    for rstd in (None, r1):
        for res in (None, dres):
            got, gw = ops.rmsnorm_bwd8(dy, p, w, EPS, rstd=rstd, dres=res)
            ref = dx if res is None else dx + res.double()
            lim = (half + 3 * FUZZ) * ref.abs() + 3 * FUZZ * terms
            if res is not None:
                lim = lim + 2.0 ** -23 * res.double().abs()
            _within("dx", got, ref, lim)
            _within("dw", gw, dw, half * dw.abs() + (FUZZ + (rows + 128) * 2.0 ** -24) * over)
            again = ops.rmsnorm_bwd8(dy, p, w, EPS, rstd=rstd, dres=res)
            assert torch.equal(got, again[0]) and torch.equal(gw, again[1])


@pytest.mark.parametrize("dtype,rows,cols,fmt", [
    (BF16, 4101, 2048, "int8"), (BF16, 3077, 4096, "e4m3"), (BF16, 4101, 1096, "e4m3"), (BF16, 2061, 8192, "int8"),
    (BF16, 3077, 512, "int8"), (FP32, 3077, 2048, "e4m3"), (FP32, 2061, 4096, "int8"), (FP32, 1029, 8192, "e4m3")])
def test_packed_norms_with_llamas_rounding_equal_those_of_the_unpacked_tensor(dtype, rows, cols, fmt):
    ops = _ops()
    x = _rows(rows, cols, 6, dtype)
    a, dy, dres = (_rows(rows, cols, s, dtype, sizes=False) for s in (7, 8, 9))
    w = (1 + randn((cols,), 10, 0.1)).to(dtype).to(DEV)
    r0, r1, r2 = (torch.empty(rows, device=DEV) for _ in range(3))
    y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, fmt, rstd=r0, llama_rounding=True)
    assert torch.equal(y, ops.rmsnorm_fwd(x, w, EPS, rstd=r1)) and torch.equal(r0, r1)
    q = ops.pack8(x, fmt)
    assert torch.equal(p.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(p.exps, q.exps)
    kept = ops.unpack8(p, dtype)
    assert torch.equal(ops.rmsnorm_fwd8(p, w, EPS, rstd=r1, llama_rounding=True), ops.rmsnorm_fwd(kept, w, EPS, rstd=r2))
    assert torch.equal(r1, r2)
    for res in (None, dres):
        for rstd in (None, r2):
            for got, ref in zip(ops.rmsnorm_bwd8(dy, p, w, EPS, rstd=rstd, dres=res, llama_rounding=True),
                                ops.rmsnorm_bwd(dy, kept, w, EPS, rstd=rstd, dres=res)):
                assert torch.equal(got, ref)
    for got, ref in zip(ops.add_rmsnorm_fwd8(p, a, w, EPS, rstd=r1, llama_rounding=True), ops.add_rmsnorm_fwd(kept, a, w, EPS, rstd=r2)):
        assert torch.equal(got, ref)
    assert torch.equal(r1, r2)


@pytest.mark.parametrize("post,pre,gate", [(True, True, "token"), (True, True, "channel"), (True, False, None), (False, True, None),
                                           (True, False, "token"), (False, True, "channel")])
@pytest.mark.parametrize("rows,cols", [(4101, 512), (4109, 1000), (2100, 2048), (1050, 4096), (530, 8192)])
def test_block_norms_in_fp32(rows, cols, post, pre, gate):
    """Forward 512 x 8, 8, 4, 2 and 1 rows a step, backward 256 times as many."""
    _check(_inputs(rows, cols, FP32, post, pre, gate, seed=21), FP32, 0.7)
