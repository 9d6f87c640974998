"""Activations in 8 bits on the GPU: storage against the oracle's (equal), the norms that
read or write it against the calls on the unpacked tensor (equal) and against fp64, and
eight_bit_checkpoint against fused_checkpoint at the kept value (equal).

Rounding counts: half a step is 2^-8 (bf16) or 2^-24 (fp32) of a value.  A row's sum of
squares runs over at most 128 terms a lane, then 6 lane steps and up to 4 waves: with the
mean, the root and the product under 144 * 2^-24 relative, a sum over rows under
(rows + 128) * 2^-24 of its terms' magnitudes.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch
from transformers.models.llama import modeling_llama as hf

from oracle import blocks as ob
from oracle import torch_llama as ot
from tests.helpers import CFG1, CFG3, hf_layer_grads, layer_weights, llama_config, load_into_hf_layer, randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FUZZ = 144 * 2.0 ** -24
FMTS = ("int8", "e4m3")
DTYPES = (torch.bfloat16, torch.float32)


def _ops():
    from femtotron_amd import ops
    return ops


def _f64(t):
    return t.detach().double().cpu().numpy()


def _stream(rows, cols, seed, dtype):
    """Rows of many sizes, some channels far above the rest."""
    x = randn((rows, cols), seed) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=torch.Generator().manual_seed(seed)).float())
    x[:, ::37] *= 300
    return x.to(dtype)


def _awkward(dtype):
    """Blocks of zeros, of the smallest and largest magnitudes, at the formats' borders, at ties, not finite."""
    x = torch.zeros(14, 72, dtype=torch.float32)
    x[1] = torch.linspace(-1, 1, 72)
    x[2, :32] = 1e-40  # below bf16's and fp32's normal numbers
    x[2, 32:] = 2.0 ** -126
    x[3] = 3.0e38
    x[3, 1::2] = -1.0e30
    x[4, 0], x[4, 1:40] = 448.0, torch.arange(39) * 0.25
    x[5, 0], x[5, 1:40] = 449.0 if dtype == torch.float32 else 450.0, torch.arange(39) * 0.25
    x[6, 0], x[6, 1:32] = 64.0, torch.arange(31) * 0.5 - 7  # ties of int8 at step 1
    x[7, 0], x[7, 1:32] = -127.75 if dtype == torch.float32 else -127.5, 0.5
    x[8, 0], x[8, 1:32] = 256.0, torch.arange(31) * 2.0 ** -10  # e4m3's subnormals and their ties
    x[9, 3], x[10, 40], x[11, 70] = float("inf"), float("-inf"), float("nan")
    x[9, 40], x[11, 0] = 3.0, 5.0
    x[12] = -0.0
    x[13] = torch.randn(72, generator=torch.Generator().manual_seed(1)) * 2.0 ** -115
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(0, 64), (1, 8), (3, 40), (7, 256), (33, 688), (5, 1000), (64, 4096), (2, 16384), (14, 72)])
def test_storage_equals_the_oracles(rows, cols, fmt, dtype):
    ops = _ops()
    x = _awkward(dtype) if rows == 14 else _stream(rows, cols, 3, dtype)
    p = ops.pack8(x.to(DEV), fmt)
    codes, exps = ob.pack8(_f64(x), fmt)
    assert p.codes.dtype == (torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
    assert np.array_equal(p.exps.cpu().numpy(), exps)
    assert np.array_equal(p.codes.float().cpu().numpy(), codes)
    for out in DTYPES:
        got = ops.unpack8(p, out)
        assert got.dtype == out and np.array_equal(_f64(got), ob.unpack8(codes, exps), equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FMTS)
def test_a_tensor_above_the_cache_is_packed_as_its_rows_are(fmt, dtype):
    ops = _ops()
    cols = 1000
    edge = (128 << 20) // (cols * dtype.itemsize)  # the last whole row below 128 MiB
    x = torch.randn(edge + 5, cols, generator=torch.Generator(DEV).manual_seed(5), device=DEV).to(dtype)
    x[:14, :72], x[-14:, -72:] = _awkward(dtype).to(DEV), _awkward(dtype).to(DEV)
    below, above = ops.pack8(x[:edge], fmt), ops.pack8(x, fmt)
    assert torch.equal(above.codes[:edge].view(torch.uint8), below.codes.view(torch.uint8))
    assert torch.equal(above.exps[:edge], below.exps)
    codes, exps = ob.pack8(_f64(x[-40:]), fmt)
    assert np.array_equal(above.exps[-40:].cpu().numpy(), exps)
    assert np.array_equal(above.codes[-40:].float().cpu().numpy(), codes)


def test_storage_takes_any_leading_shape_and_refuses_what_it_cannot_read():
    ops = _ops()
    x = randn((2, 3, 64), 4).bfloat16().to(DEV)
    p = ops.pack8(x)
    assert p.codes.shape == (2, 3, 64) and p.exps.shape == (2, 3, 2)
    assert torch.equal(ops.unpack8(p), ops.unpack8(ops.pack8(x.view(6, 64))).view(2, 3, 64))
    with pytest.raises(ValueError, match="contiguous"):
        ops.pack8(x.transpose(0, 1))
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.pack8(x[..., :60].contiguous())
    with pytest.raises(TypeError, match="float16"):
        ops.pack8(x.half())
    with pytest.raises(ValueError, match="one of"):
        ops.pack8(x, "e5m2")
    with pytest.raises(ValueError, match="exps"):
        ops.unpack8(ops.Packed8(p.codes, p.exps[:, :, :1].contiguous()))
    with pytest.raises(TypeError, match="codes"):
        ops.unpack8(ops.Packed8(p.codes.short(), p.exps))
    with pytest.raises(TypeError, match="float16"):
        ops.unpack8(p, torch.float16)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="last dim"):
        ops.rmsnorm_fwd8(p, w[:32], EPS)
    with pytest.raises(ValueError, match="shape"):
        ops.add_rmsnorm_fwd8(p, x[:1], w, EPS)
    with pytest.raises(TypeError, match="mismatch"):
        ops.rmsnorm_bwd8(x.float(), p, w, EPS)
    with pytest.raises(ValueError, match="rstd"):
        ops.rmsnorm_fwd8(p, w, EPS, rstd=torch.empty(5, device=DEV))
    from femtotron_amd._lib import FemtoHipError
    odd = torch.empty(6 * 64 + 8, dtype=torch.bfloat16, device=DEV)[4:4 + 6 * 64].view(6, 64)
    with pytest.raises(FemtoHipError, match="aligned"):
        ops.pack8(odd)


CASES = [(1, 8), (7, 256), (33, 688), (5, 1000), (130, 2048), (2050, 1024), (9, 4096), (2100, 4096), (3, 8192)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", CASES)
def test_norms_equal_those_of_the_unpacked_tensor(rows, cols, fmt, dtype):
    ops = _ops()
    x = _stream(rows, cols, 5, dtype).to(DEV)
    a, dy, dres = (randn((rows, cols), s).to(dtype).to(DEV) for s in (6, 7, 8))
    w = (1 + randn((cols,), 9, 0.1)).to(dtype).to(DEV)
    r0, r1, r2 = (torch.empty(rows, device=DEV) for _ in range(3))
    y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, fmt, rstd=r0, llama_rounding=True)
    assert torch.equal(y, ops.rmsnorm_fwd(x, w, EPS, rstd=r1)) and torch.equal(r0, r1)
    q = ops.pack8(x, fmt)
    assert torch.equal(p.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(p.exps, q.exps)
    kept = ops.unpack8(p, dtype)
    assert torch.equal(ops.rmsnorm_fwd8(p, w, EPS, rstd=r1, llama_rounding=True), ops.rmsnorm_fwd(kept, w, EPS, rstd=r2)) and torch.equal(r1, r2)
    for got, ref in zip(ops.add_rmsnorm_fwd8(p, a, w, EPS, rstd=r1, llama_rounding=True), ops.add_rmsnorm_fwd(kept, a, w, EPS, rstd=r2)):
        assert torch.equal(got, ref)
    assert torch.equal(r1, r2)
    ops.rmsnorm_fwd8(p, w, EPS, rstd=r1, llama_rounding=True)
    for rstd in (None, r1):
        for res in (None, dres):
            for got, ref in zip(ops.rmsnorm_bwd8(dy, p, w, EPS, rstd=rstd, dres=res, llama_rounding=True),
                                ops.rmsnorm_bwd(dy, kept, w, EPS, rstd=rstd, dres=res)):
                assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1, 8), (33, 688), (300, 2048), (40, 4096)])
def test_norms_against_fp64(rows, cols, fmt, dtype):
    ops = _ops()
    x = _stream(rows, cols, 10, dtype)
    a, dy, dres = (randn((rows, cols), s).to(dtype) for s in (11, 12, 13))
    w = (1 + randn((cols,), 14, 0.1)).to(dtype)
    xd, ad, dyd, dresd, wd = (t.to(DEV) for t in (x, a, dy, dres, w))
    half = HALF[dtype]
    kept = ob.unpack8(*ob.pack8(_f64(x), fmt))
    for llama in (False, True):
        # y is rounded once; with llama_rounding its normalised value was rounded too
        inner = half if llama else 0.0
        tol = half + inner * (1 + half) + FUZZ
        y, p = ops.rmsnorm_fwd_pack8(xd, wd, EPS, fmt, llama_rounding=llama)
        ref = ob.rmsnorm(_f64(x), _f64(w), EPS)
        assert (np.abs(_f64(y) - ref) <= tol * np.abs(ref)).all()
        ref = ob.rmsnorm(kept, _f64(w), EPS)
        assert (np.abs(_f64(ops.rmsnorm_fwd8(p, wd, EPS, llama_rounding=llama)) - ref) <= tol * np.abs(ref)).all()
        h, z = ops.add_rmsnorm_fwd8(p, ad, wd, EPS, llama_rounding=llama)
        s = kept + _f64(a)
        assert (np.abs(_f64(h) - s) <= (half + 2.0 ** -24) * np.abs(s)).all()
        ref = ob.rmsnorm(_f64(h), _f64(w), EPS)
        assert (np.abs(_f64(z) - ref) <= tol * np.abs(ref)).all()
        dx, dw = ops.rmsnorm_bwd8(dyd, p, wd, EPS, dres=dresd, llama_rounding=llama)
        rdx, rdw, terms = ob.rmsnorm_bwd(_f64(dy), kept, _f64(w), EPS)
        rdx = rdx + _f64(dres)
        # with llama_rounding dy w is rounded, in dx's own term and in the mean; the sum is rounded once
        lim = (half + 3 * FUZZ) * np.abs(rdx) + (inner + 3 * FUZZ) * terms + 2.0 ** -23 * np.abs(_f64(dres))
        assert (np.abs(_f64(dx) - rdx) <= lim).all()
        # and the normalised value before the sum over rows, which is rounded once
        n = np.abs(_f64(dy) * ob.rmsnorm(kept, 1.0, EPS)).sum(0)
        assert (np.abs(_f64(dw) - rdw) <= half * np.abs(rdw) + (inner + FUZZ + (rows + 128) * 2.0 ** -24) * n).all()


def test_gradient_is_the_slope_of_the_norm_at_the_kept_value():
    """fp32: <dx, d> against a difference of sum(dy norm(x^ + t d)) in fp64, and dw's."""
    ops = _ops()
    x, dy, d = (randn((6, 200), s) for s in (15, 16, 17))
    w, dwdir = 1 + randn((200,), 18, 0.1), randn((200,), 19)
    p = ops.pack8(x.to(DEV), "int8")
    dx, dw = ops.rmsnorm_bwd8(dy.to(DEV), p, w.to(DEV), EPS)
    kept, t = _f64(ops.unpack8(p, torch.float32)), 1e-5

    def f(s):
        return (_f64(dy) * ob.rmsnorm(kept + s * _f64(d), _f64(w) + s * _f64(dwdir), EPS)).sum()

    slope = (f(t) - f(-t)) / (2 * t)
    got = (_f64(dx) * _f64(d)).sum() + (_f64(dw) * _f64(dwdir)).sum()
    _, _, terms = ob.rmsnorm_bwd(_f64(dy), kept, _f64(w), EPS)
    n = np.abs(_f64(dy) * ob.rmsnorm(kept, 1.0, EPS)).sum(0)
    lim = ((3 * FUZZ + 2.0 ** -24) * (terms + np.abs(_f64(dx))) * np.abs(_f64(d))).sum()
    lim += ((FUZZ + 134 * 2.0 ** -24) * n * np.abs(_f64(dwdir))).sum()
    # the difference itself: t^2 times a third derivative (under 1e4), and 2^-52 of its 1200 terms over t
    assert abs(got - slope) <= lim + 1e-10 * 1e4 + 1200 * 2.0 ** -52 / t * 10


def test_rows_that_hold_nothing_finite_or_nothing_at_all():
    ops = _ops()
    x = _awkward(torch.bfloat16).to(DEV)
    w = torch.ones(72, dtype=torch.bfloat16, device=DEV)
    y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, "int8")
    assert torch.equal(y.isnan(), ops.rmsnorm_fwd(x, w, EPS).isnan())
    z = ops.rmsnorm_fwd8(p, w, EPS)
    assert bool(z[9:12].isnan().all()) and bool(z[[0, 1, 2, 4, 5, 6, 7, 8, 12]].isfinite().all())
    assert torch.count_nonzero(z[0]) == 0 and torch.count_nonzero(z[12]) == 0
    dx, dw = ops.rmsnorm_bwd8(torch.ones_like(x), p, w, EPS)
    assert bool(dx[9:12].isnan().all()) and bool(dx[[0, 1, 4, 12]].isfinite().all()) and bool(dw.isnan().any())
    e = ops.pack8(x[:0])
    dx, dw = ops.rmsnorm_bwd8(x[:0], e, w, EPS)
    assert dx.shape == (0, 72) and torch.count_nonzero(dw) == 0
    assert ops.rmsnorm_fwd8(e, w, EPS).shape == (0, 72) and ops.unpack8(e).shape == (0, 72)


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last rows equal those packed alone."""
    ops = _ops()
    rows, cols = (1 << 20) + 3, 4096 + 8
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    tail = randn((5, cols), 20).bfloat16().to(DEV)
    x[-5:] = tail
    p, q = ops.pack8(x, "int8"), ops.pack8(tail, "int8")
    assert torch.equal(p.codes[-5:], q.codes) and torch.equal(p.exps[-5:], q.exps)
    x.zero_()
    x = ops.unpack8(p)
    assert torch.equal(x[-5:], ops.unpack8(q))


def test_another_stream_and_a_replayed_graph():
    """Captured and replayed with new inputs, other work between the replays."""
    ops = _ops()
    w = (1 + randn((2048,), 21, 0.1)).bfloat16().to(DEV)
    x, dy = (torch.empty(300, 2048, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def step():
        y, p = ops.rmsnorm_fwd_pack8(x, w, EPS, "e4m3")
        return (y, ops.rmsnorm_fwd8(p, w, EPS), *ops.rmsnorm_bwd8(dy, p, w, EPS, dres=x), ops.unpack8(p))

    side = torch.cuda.Stream()
    x.copy_(randn(x.shape, 22)), dy.copy_(randn(x.shape, 23))
    ref = step()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for k in range(4):
        x.copy_(randn(x.shape, 30 + k)), dy.copy_(randn(x.shape, 40 + k))
        g.replay()
        torch.cuda.synchronize()
        ref = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref)), k


# ------------------------------------------------------------------ eight_bit_checkpoint
def _layer_step(c, dtype, B, S, fn, x):
    from femtotron_amd.training import ActivationCheckpointWrapper
    layer = hf.LlamaDecoderLayer(llama_config(c, layers=1), layer_idx=0)
    load_into_hf_layer(layer, layer_weights(c, seed=42, norm_mean=1.0))
    layer = layer.to(device=DEV, dtype=dtype)
    cos, sin = ot.rope_cos_sin(S, c["hidden"] // c["heads"], c["theta"], dtype, device=DEV)
    x = x.clone().requires_grad_(True)
    out = ActivationCheckpointWrapper(layer, checkpoint_fn=fn)(
        x, attention_mask=None, position_embeddings=(cos, sin), past_key_values=None, use_cache=False)
    out.backward(randn((B, S, c["hidden"]), 44).to(device=DEV, dtype=dtype))
    return out.detach(), {"x": x.grad, **hf_layer_grads(layer)}


@pytest.mark.parametrize("one_call", [True, False])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("c,dtype,B,S", [(CFG1, torch.bfloat16, 2, 128), (CFG1, torch.float32, 2, 77), (CFG3, torch.bfloat16, 1, 333)])
def test_layer_is_the_fused_layer_at_the_kept_value(c, dtype, B, S, fmt, one_call, monkeypatch):
    from femtotron_amd import dispatch_counts, eight_bit_checkpoint, fused_checkpoint, fused_layer, reset_dispatch_counts
    ops = _ops()
    if not one_call:
        monkeypatch.setattr(fused_layer, "ONE_CALL_MAX_BYTES", 0)
    x = randn((B, S, c["hidden"]), 43).to(device=DEV, dtype=dtype)
    reset_dispatch_counts()
    out, grads = _layer_step(c, dtype, B, S, eight_bit_checkpoint(fmt), x)
    assert dispatch_counts() == {"fused": 1, "fallback": 0}
    ref, _ = _layer_step(c, dtype, B, S, fused_checkpoint, x)
    assert torch.equal(out, ref)
    _, at_kept = _layer_step(c, dtype, B, S, fused_checkpoint, ops.unpack8(ops.pack8(x, fmt), dtype))
    for k, g in grads.items():
        assert torch.equal(g, at_kept[k]), k


@pytest.mark.parametrize("fmt", FMTS)
def test_selective_modules_are_the_fused_ones_at_the_kept_value(fmt):
    from femtotron_amd import eight_bit_checkpoint, fused_checkpoint
    ops = _ops()
    layer = hf.LlamaDecoderLayer(llama_config(CFG1, layers=1), 0)
    load_into_hf_layer(layer, layer_weights(CFG1, seed=42, norm_mean=1.0))
    layer = layer.to(DEV, torch.bfloat16)
    x = randn((2, 100, 256), 50).bfloat16().to(DEV)
    dy = randn((2, 100, 256), 51).bfloat16().to(DEV)
    for mod in (layer.mlp, layer.input_layernorm):
        def step(fn, at):
            leaf = at.clone().requires_grad_(True)
            y = fn(mod, leaf, use_reentrant=False)
            return y.detach(), torch.autograd.grad(y, [leaf, *mod.parameters()], dy)
        y, grads = step(eight_bit_checkpoint(fmt), x)
        assert torch.equal(y, step(fused_checkpoint, x)[0])
        for a, b in zip(grads, step(fused_checkpoint, ops.unpack8(ops.pack8(x, fmt)))[1]):
            assert torch.equal(a, b)
        with torch.no_grad():
            assert torch.equal(eight_bit_checkpoint(fmt)(mod, x, use_reentrant=False), y)


def test_a_model_keeps_half_and_learns_the_same_way():
    """A model's step: the loss is fused_checkpoint's bit for bit, what its layers keep is
    33/64 of it, and its gradient points the same way.  With each layer's input off by at
    most 2^-7 of its block's largest element (rms under 0.9% of an N(0, 1) block: a step of
    2^-6 to 2^-5 of the largest, uniform, over sqrt(12)), two layers' gradients are off by a few
    times that: under 10%, so a cosine of at least 1 - 0.1^2 / 2."""
    from femtotron_amd import eight_bit_checkpoint, fused_checkpoint
    from femtotron_amd.model import build_llama_model, init_llama_weights_
    from femtotron_amd.scripts.presets import get_ac_policy
    from femtotron_amd.training import apply_activation_checkpointing
    ids = torch.randint(0, CFG3["vocab"], (2, 2048), generator=torch.Generator().manual_seed(7)).to(DEV)
    got = {}
    for name, fn in (("16", fused_checkpoint), ("8", eight_bit_checkpoint("int8"))):
        model = init_llama_weights_(build_llama_model(llama_config(CFG3, layers=2)), device=DEV, dtype=torch.bfloat16, seed=3)
        apply_activation_checkpointing(model, get_ac_policy("llama_decoder_layer"), checkpoint_fn=fn)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        hidden = model.model(ids)
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated() - before
        del hidden
        loss = model(ids, labels=ids, materialize_logits=False)["loss"]
        loss.backward()
        got[name] = loss.detach(), held, torch.cat([p.grad.float().flatten() for p in model.model.layers.parameters()])
        del model, loss
    assert torch.equal(got["16"][0], got["8"][0])
    T, H = ids.numel(), CFG3["hidden"]
    # two layers' inputs; everything else that is held is the same
    assert got["16"][1] - got["8"][1] == 2 * (2 * T * H - T * H - T * H // 32)
    a, b = got["16"][2].double(), got["8"][2].double()
    assert float((a @ b) / (a.norm() * b.norm())) > 1 - 0.1 ** 2 / 2
