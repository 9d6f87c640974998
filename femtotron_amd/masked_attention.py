"""Attention of documents packed into rows: under document, prefix and window masks, with
capped scores and biases by distance, differentiable; and over a cache, for answers.

The stock layer's attention (transformers 5.15.0, models/llama/modeling_llama.py:235-281;
``ops.attn_fwd``) is causal over whole rows with a plain softmax.  Rows that hold several
documents, or a prompt that all of its document sees, or padding, need

    o_i = sum_j softmax_j(z_ij) v_j,   z_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i - j|

over the j that token i sees, which ``attention_mask`` says.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import ops


class AttentionMask:
    """What each token of a batch sees (``attention_mask``): one for all layers of a step."""

    __slots__ = ("table", "batch", "seq_len")

    def __init__(self, table: torch.Tensor, batch: int, seq_len: int):
        self.table, self.batch, self.seq_len = table, batch, seq_len

    def __repr__(self) -> str:
        return f"AttentionMask(batch={self.batch}, seq_len={self.seq_len}, device={self.table.device})"


def attention_mask(batch: int, seq_len: int, starts: torch.Tensor | None = None, lengths: torch.Tensor | None = None, *,
                   prefix: torch.Tensor | None = None, window: int | None = None, causal: bool = True,
                   device: torch.device | str | None = None) -> AttentionMask:
    """The mask of ``masked_attention`` for [batch, seq_len] tokens, counted row by row (token
    s of row b is b * seq_len + s).

    Document d is the lengths[d] tokens from starts[d] on (int64 vectors on the device, starts
    ascending; packed sequences: starts = cu_seqlens[:-1]); without ``lengths`` each ends
    where the next begins, and one that runs into the next ends there in any case.  Without
    ``starts`` each row is one document, of its first lengths[b] tokens.  A token sees its own
    document: what is up to itself (``causal``) or all of it; with ``prefix`` (int64, one a
    document; causal) also the document's first prefix[d] tokens; with ``window`` what is less
    than window tokens away (without a prefix).  A token of no document sees nothing: its
    output and its gradients are 0.

    The values stay on the device and are not waited for: starts that do not ascend are not
    refused, and give some mask within the rows."""
    if batch < 0 or seq_len < 0:
        raise ValueError(f"attention_mask: batch and seq_len must not be negative, got {batch}, {seq_len}")
    if window is not None and window < 1:
        raise ValueError(f"attention_mask: window must be at least 1, got {window}")
    if prefix is not None and (window is not None or not causal):
        raise ValueError("attention_mask: a prefix goes with causal and without a window")
    given = next((t for t in (starts, lengths, prefix) if t is not None), None)
    if device is None:
        device = torch.device("cuda") if given is None else given.device
    else:
        device = torch.device(device)
        if given is not None and device.index is not None and device != given.device:
            raise ValueError(f"attention_mask: a tensor on {given.device}, the mask on {device}")
        device = device if given is None else given.device
    if device.type != "cuda":
        raise ValueError("femtohip ops take HIP device tensors only")
    starts, lengths, prefix = (None if t is None else t.contiguous() for t in (starts, lengths, prefix))
    table = ops.attn_mask(batch * seq_len, seq_len, starts, lengths, prefix, window or 0, causal, device)
    return AttentionMask(table, batch, seq_len)


def _laid_out(t: torch.Tensor, seq_len: int) -> tuple[torch.Tensor, int]:
    """t as token rows that the kernels read (itself, or a copy), and their row stride."""
    ld = ops.token_rows(t, seq_len)
    if ld:
        return t, ld
    return ops.aligned(t), t.size(-1)


class MaskedAttentionFunction(torch.autograd.Function):
    """Saved: q, k, v, o (bf16: and 8 more bits of it) and an fp32 value a token and head."""

    @staticmethod
    def forward(ctx, q, k, v, table, slopes, args, seq_len):
        o, lse, low = ops.masked_attn_fwd_checked(args, q, k, v, table, slopes, True)
        ctx.save_for_backward(q, k, v, o, lse, low, slopes)
        ctx.table, ctx.args, ctx.seq_len = table, args, seq_len  # the table is the step's, not the layer's
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, low, slopes = ctx.saved_tensors
        # autograd hands the gradient in of the output's shape, dtype and device
        do, lddo = _laid_out(do, ctx.seq_len)
        return (*ops.masked_attn_bwd_checked(ctx.args, q, k, v, o, do, lddo, lse, low, ctx.table, slopes), None, None, None, None)


def _score(name: str, head_dim: int, scale: float | None, cap: float | None,
           slopes: torch.Tensor | None) -> tuple[float, float]:
    """(scale, cap) as the kernels take them, 0 for no cap."""
    for v, n in ((scale, "scale"), (cap, "cap"), (slopes, "slopes")):
        if v is not None and ops.wants_derivative(v):
            raise TypeError(f"{name}: {n} is a constant and gets no gradient")
    if head_dim not in (32, 64, 128):
        raise ValueError(f"{name}: head_dim must be 32, 64 or 128, got {head_dim}")
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"{name}: scale must be positive, got {scale}")
    if cap is None:
        return scale, 0.0
    cap32 = ctypes.c_float(cap).value  # the kernels', for which 0 is no cap
    if not 0 < cap32 < math.inf:
        raise ValueError(f"{name}: cap must be positive and finite in fp32, or None, got {cap}")
    return scale, cap32


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, *, head_dim: int,
                     scale: float | None = None, cap: float | None = None,
                     slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [batch, seq, heads * head_dim] (or [tokens, ...]) over k and v of the same
    tokens and kv heads * head_dim columns (query head h reads kv head h * kv heads // heads;
    column views of a packed projection are read in place), each token over what ``mask`` lets
    it see; differentiable in q, k and v (once, and in reverse mode).

    head_dim 32, 64 or 128; ``scale`` (None: head_dim ** -0.5) on the products; ``cap``: scores
    become cap * tanh(score / cap) (a cap of at most 2^126 times the scale, in bf16 of at most 4096); ``slopes`` (fp32, one a
    query head): less slopes[h] times the distance, after the cap.  bf16 or fp32 on a HIP
    device.  Nothing that a token does not see reaches it, infinities and NaN included."""
    scale, cap = _score("masked_attention", head_dim, scale, cap, slopes)
    seq_len = mask.seq_len
    tokens = mask.batch * seq_len
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        shape = t.shape
        if not (len(shape) == 3 and shape[0] == mask.batch and shape[1] == seq_len or len(shape) == 2 and shape[0] == tokens):
            raise ValueError(f"masked_attention: {n} must be [{mask.batch}, {seq_len}, heads * head_dim] or "
                             f"[{tokens}, heads * head_dim] under this mask, got {tuple(shape)}")
    dt, nh, nkv = ops.masked_attn_check("masked_attention", q, k, v, mask.table, slopes, tokens, head_dim)
    (q, ldq), (k, ldk), (v, ldv) = _laid_out(q, seq_len), _laid_out(k, seq_len), _laid_out(v, seq_len)
    args = (dt, ldq, ldk, ldv, tokens, nh, nkv, head_dim, scale, cap)
    if ops.differentiated(q, k, v):
        return MaskedAttentionFunction.apply(q, k, v, mask.table, slopes, args, seq_len)
    return ops.masked_attn_fwd_checked(args, q, k, v, mask.table, slopes, False)[0]


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *, head_dim: int,
                    scale: float | None = None, cap: float | None = None, slopes: torch.Tensor | None = None,
                    window: int | None = None) -> torch.Tensor:
    """Attention of the newest tokens of each sequence, q [batch, new, heads * head_dim], over
    a cache of the sequences' keys and values, [batch, room, kv heads * head_dim] or [batch,
    room, kv heads, head_dim] (a view: a cache laid out [batch, kv heads, room, head_dim] goes
    in transposed), the new tokens' own among them.  Sequence b holds lengths[b] (int64 on the
    device, taken within 0 and room); its token u stands at place lengths[b] - new + u and
    sees the places up to its own, with ``window`` the last window of them.  A token before
    place 0 gets 0.  No place from lengths[b] on is read.

    Scores as in ``masked_attention``, distances between places.  Without derivatives: refused
    where one is asked for."""
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        if ops.wants_derivative(t):
            raise TypeError(f"cache_attention has no derivatives, and {n} wants one (use it under torch.no_grad())")
    scale, cap = _score("cache_attention", head_dim, scale, cap, slopes)
    if window is not None and window < 1:
        raise ValueError(f"cache_attention: window must be at least 1, got {window}")
    if q.dim() != 3:
        raise ValueError(f"cache_attention: q must be [batch, new, heads * head_dim], got {tuple(q.shape)}")
    q, ldq = _laid_out(q, q.shape[1])
    return ops.cache_attn(q, ldq, k_cache, v_cache, lengths.contiguous(), head_dim=head_dim, scale=scale, cap=cap,
                          slopes=slopes, window=window or 0)
