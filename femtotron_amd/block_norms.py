"""The norms after and before a block, with the block's gate and residual scale, as one
differentiable call.

A stock Llama layer adds a block's output to the residual stream and norms the sum for
the next block (transformers 5.15.0, models/llama/modeling_llama.py:284-325;
``ops.add_rmsnorm_fwd``).  Layers that also norm the block's output, gate it or scale it
before the add need

    h = x + scale * gate * RMSNorm(a; w_post)      y = RMSNorm(h; w_pre)

whose forward and backward each run in one pass here (fh_block_norms_fwd / _bwd).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class BlockNormsFunction(torch.autograd.Function):
    """Saved: a, h, the vectors and the gate, and two fp32 values a row."""

    @staticmethod
    def forward(ctx, args, x, a, w_post, w_pre, gate, scale, eps):
        rows = args[2]
        rstd_post = None if w_post is None else x.new_empty(rows, dtype=torch.float32)
        rstd_pre = None if w_pre is None else x.new_empty(rows, dtype=torch.float32)
        h, y = ops.block_norms_fwd_checked(args, x, a, w_post, w_pre, gate, scale, eps, rstd_post, rstd_pre)
        ctx.save_for_backward(None if w_pre is None else h, a if w_post is not None or gate is not None else None, w_post,
                              w_pre, gate, rstd_post, rstd_pre)
        ctx.args, ctx.scale = args, scale
        ctx.set_materialize_grads(False)
        return h, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dy):
        if dh is None and dy is None:
            return (None,) * 8
        h, a, w_post, w_pre, gate, rstd_post, rstd_pre = ctx.saved_tensors
        dh, dy = ops.aligned(dh), ops.aligned(dy)
        if dh is None:
            dh = torch.zeros_like(dy)
        if dy is None and w_pre is not None:
            dy = torch.zeros_like(dh)
        # autograd hands gradients in of the outputs' shape, dtype and device
        return (None, *ops.block_norms_bwd_checked(ctx.args, dh, dy, h, a, w_post, w_pre, gate, ctx.scale, rstd_post,
                                                   rstd_pre), None, None)


def block_norms(x: torch.Tensor, a: torch.Tensor, w_post: torch.Tensor | None = None,
                w_pre: torch.Tensor | None = None, *, gate: torch.Tensor | None = None, scale: float = 1.0,
                eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(h, y) = (x + scale * gate * RMSNorm(a; w_post), RMSNorm(h; w_pre)) over the last
    dim of x and a (one shape, bf16 or fp32, on a HIP device), differentiable in every
    tensor (once, and in reverse mode).

    ``w_post`` None: a enters without a norm; ``w_pre`` None: y is None (one of the
    two is given).  ``gate``: one value a channel ([hidden], or with leading ones), one an
    element (x's shape: expand a gate that is shared along some dims), or None.
    y is the norm of h in x's dtype, as returned.  ``scale`` is a number: a learned one
    belongs in the gate."""
    if isinstance(scale, torch.Tensor) and (scale.requires_grad or ops.wants_derivative(scale)):
        raise TypeError("block_norms: scale is a number and gets no gradient; fold a learned one into the gate")
    if gate is not None and gate.shape != x.shape and gate.numel() == x.shape[-1] == gate.shape[-1]:
        gate = gate.reshape(-1)
    tensors = tuple(map(ops.aligned, (x, a, w_post, w_pre, gate)))
    if ops.differentiated(*tensors):
        return BlockNormsFunction.apply(ops.block_norms_check("block_norms", *tensors), *tensors, float(scale), float(eps))
    x, a, w_post, w_pre, gate = tensors
    return ops.block_norms_fwd(x, a, w_post, w_pre, float(eps), gate=gate, scale=float(scale))
