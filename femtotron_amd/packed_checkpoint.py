"""Checkpointed modules that keep their input in 8 bits.

What activation checkpointing holds from the forward to the backward is one input
per checkpointed module (torch.utils.checkpoint's ``_NoopSaveInputs``,
torch/utils/checkpoint.py:794-831, under femtotron/training/activation_ckpt.py:78-86).
These autograd nodes are those of fused_layer.py and fused_parts.py with that input
kept as ``ops.Packed8``: 8.25 bits an element instead of 16 or 32.

The forward computes from the input itself, so outputs and losses are those of
``fused_checkpoint`` bit for bit.  The backward is that of ``fused_checkpoint`` at
the kept value x^, again bit for bit.  With m the largest magnitude of x's block of
32, |x^ - x| is at most the larger of 2^-7 m and 2^-119 in "int8", and of 2^-4 |x|, 2^-17 m
and 2^-128 in "e4m3".

* decoder layer: the first norm's pass packs x; in the backward the recompute's
  norm and residual add + norm and the norm's backward read the codes, and x^ is
  not laid out (small layers that run as one native call unpack it first);
* RMSNorm: packed by the forward's pass, read by the backward kernel;
* MLP: x^ is laid out for the backward's products, whose operand it is.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from .fused_layer import _one_call, _one_call_backward, layer_backward, layer_forward
from .fused_parts import mlp_backward, mlp_forward
from .projections import count_hand


class PackedDecoderLayerFunction(torch.autograd.Function):
    """FusedDecoderLayerFunction whose input is kept in 8 bits."""

    @staticmethod
    def forward(ctx, fmt, x, cos, sin, shp, wq, wk, wv, wo, wg, wu, wd, w1, w2):
        B, S, H = x.shape
        w = (wq, wk, wv, wo, wg, wu, wd, w1, w2)
        x2 = x.reshape(B * S, H)
        call = _one_call(x, cos, sin, shp, w)
        if call is not None:
            out = ops.layer_fwd(call[0], call[1], x)
            count_hand(4)
            kept = ops.pack8(x2, fmt)
        else:
            out, kept = layer_forward(x2, cos, sin, shp, B, S, w, keep=False, pack=fmt)
        ctx.save_for_backward(*kept, cos, sin, *w)
        ctx.shp, ctx.batch, ctx.seq = shp, B, S
        return out.view(B, S, H)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        codes, exps, cos, sin, *w = ctx.saved_tensors
        B, S = ctx.batch, ctx.seq
        dx, dws = _backward(ops.aligned(dout), ops.Packed8(codes, exps), cos, sin, ctx.shp, B, S, tuple(w))
        return (None, dx.view(B, S, codes.shape[-1]), None, None, None, *dws)


def _backward(dout, kept, cos, sin, shp, B, S, w):
    T, H = kept.codes.shape
    # Whether the layer runs as one call goes by sizes, weights and dout, which stands
    # for the x of its shape and dtype that is not laid out yet.
    call = _one_call(dout, cos, sin, shp, w, dout)
    if call is not None:
        return _one_call_backward(call, ops.unpack8(kept, dout.dtype).view(B, S, H), dout, shp, w)
    acts = layer_forward(kept, cos, sin, shp, B, S, w, keep=True)
    return layer_backward(dout.view(T, H), kept, cos, sin, shp, B, S, w, acts)


class PackedMLPFunction(torch.autograd.Function):
    """FusedMLPFunction whose input is kept in 8 bits."""

    @staticmethod
    def forward(ctx, fmt, z, wg, wu, wd):
        z2 = z.reshape(-1, z.shape[-1])
        m = mlp_forward(z2, wg, wu, wd, keep=False)
        ctx.save_for_backward(*ops.pack8(z2, fmt), wg, wu, wd)
        return m.view(z.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dm):
        codes, exps, wg, wu, wd = ctx.saved_tensors
        z2 = ops.unpack8(ops.Packed8(codes, exps), dm.dtype)
        dz, dwg, dwu, dwd = mlp_backward(ops.aligned(dm).view(-1, z2.shape[-1]), z2, wg, wu, wd,
                                         mlp_forward(z2, wg, wu, wd, keep=True))
        return None, dz.view(dm.shape), dwg, dwu, dwd


class PackedRMSNormFunction(torch.autograd.Function):
    """FusedRMSNormFunction whose input is kept in 8 bits."""

    @staticmethod
    def forward(ctx, fmt, x, w, eps):
        y, kept = ops.rmsnorm_fwd_pack8(x, w, eps, fmt, llama_rounding=True)
        ctx.save_for_backward(*kept, w)
        ctx.eps = eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, exps, w = ctx.saved_tensors
        dx, dw = ops.rmsnorm_bwd8(ops.aligned(dy), ops.Packed8(codes, exps), w, ctx.eps, llama_rounding=True)
        return None, dx, dw, None
