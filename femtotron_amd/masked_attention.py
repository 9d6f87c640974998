"""Attention of documents packed into rows: under document, prefix and window masks, with
capped scores and biases by distance, differentiable; and over a cache, for answers.

The stock layer's attention (transformers 5.15.0, models/llama/modeling_llama.py:235-281;
``ops.attn_fwd``) is causal over whole rows with a plain softmax.  Rows that hold several
documents, or a prompt that all of its document sees, or padding, need

    o_i = sum_j softmax_j(z_ij) v_j,   z_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i - j|

over the j that token i sees, which ``attention_mask`` says.
"""
from __future__ import annotations

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
    for t in (starts, lengths, prefix):
        if t is not None:
            if device is not None and torch.device(device) != t.device and torch.device(device).index is not None:
                raise ValueError(f"attention_mask: a tensor on {t.device}, the mask on {device}")
            device = t.device
    if device is None:
        device = torch.device("cuda")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("femtohip ops take HIP device tensors only")
    starts, lengths, prefix = (None if t is None else t.contiguous() for t in (starts, lengths, prefix))
    table = ops.attn_mask(batch * seq_len, seq_len, starts, lengths, prefix, window or 0, causal, device)
    return AttentionMask(table, batch, seq_len)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as token rows that the kernels read in place, laid out first where it is none."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    ld, unit = t.stride()
    if (unit == 1 or t.shape[1] == 1) and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (ld >= t.shape[1] and ld % 8 == 0)):
        return t
    return ops.aligned(t)


class MaskedAttentionFunction(torch.autograd.Function):
    """Saved: q, k, v, o (bf16: and 8 more bits of it) and an fp32 value a token and head."""

    @staticmethod
    def forward(ctx, q, k, v, table, slopes, how):
        rows = _rows(q), _rows(k), _rows(v)
        o, lse, low = ops.masked_attn_fwd(*rows, table, slopes=slopes, **how)
        ctx.save_for_backward(*rows, o, lse, low, table, slopes)
        ctx.how, ctx.shapes = how, (q.shape, k.shape, v.shape)
        return o.view(q.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, low, table, slopes = ctx.saved_tensors
        grads = ops.masked_attn_bwd(q, k, v, o, _rows(do), lse, low, table, slopes=slopes, **ctx.how)
        return (*(g.view(s) for g, s in zip(grads, ctx.shapes)), None, None, None)


def _score(name: str, head_dim: int, scale: float | None, cap: float | None, slopes: torch.Tensor | None) -> dict:
    for v, n in ((scale, "scale"), (cap, "cap"), (slopes, "slopes")):
        if ops.wants_derivative(v):
            raise TypeError(f"{name}: {n} is a constant and gets no gradient")
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError(f"{name}: scale must be positive, got {scale}")
    if cap is not None and not 0 < cap < float("inf"):
        raise ValueError(f"{name}: cap must be positive, or None, got {cap}")
    return dict(head_dim=head_dim, scale=scale, cap=float(cap or 0.0))


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, *, head_dim: int,
                     scale: float | None = None, cap: float | None = None,
                     slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [batch, seq, heads * head_dim] (or [tokens, ...]) over k and v of the same
    tokens and kv heads * head_dim columns (query head h reads kv head h * kv heads // heads;
    column views of a packed projection are read in place), each token over what ``mask`` lets
    it see; differentiable in q, k and v (once, and in reverse mode).

    head_dim 32, 64 or 128; ``scale`` (None: head_dim ** -0.5) on the products; ``cap``: scores
    become cap * tanh(score / cap); ``slopes`` (fp32, one a query head): less slopes[h] times
    the distance, after the cap.  bf16 or fp32 on a HIP device.  Nothing that a token does not
    see reaches it, infinities and NaN included."""
    how = _score("masked_attention", head_dim, scale, cap, slopes)
    tokens = mask.batch * mask.seq_len
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() not in (2, 3) or t.numel() != tokens * t.shape[-1] or (t.dim() == 3 and t.shape[1] != mask.seq_len):
            raise ValueError(f"masked_attention: {n} must be [{mask.batch}, {mask.seq_len}, heads * head_dim] or "
                             f"[{tokens}, heads * head_dim] under this mask, got {tuple(t.shape)}")
    if ops.differentiated(q, k, v):
        return MaskedAttentionFunction.apply(q, k, v, mask.table, slopes, how)
    o, _, _ = ops.masked_attn_fwd(_rows(q), _rows(k), _rows(v), mask.table, slopes=slopes, need_grad=False, **how)
    return o.view(q.shape)


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
    how = _score("cache_attention", head_dim, scale, cap, slopes)
    if window is not None and window < 1:
        raise ValueError(f"cache_attention: window must be at least 1, got {window}")
    if q.dim() != 3:
        raise ValueError(f"cache_attention: q must be [batch, new, heads * head_dim], got {tuple(q.shape)}")
    caches = []
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dim() == 3 and head_dim > 0 and t.shape[-1] % head_dim == 0:
            t = t.unflatten(-1, (t.shape[-1] // head_dim, head_dim))
        if t.dim() != 4 or t.shape[0] != q.shape[0] or t.shape[3] != head_dim:
            raise ValueError(f"cache_attention: {n} must be [{q.shape[0]}, room, kv heads * {head_dim}] or "
                             f"[{q.shape[0]}, room, kv heads, {head_dim}], got {tuple(t.shape)}")
        caches.append(t)
    del how["head_dim"]
    o = ops.cache_attn(_rows(q), *caches, lengths.contiguous(), n_new=q.shape[1], slopes=slopes, window=window or 0, **how)
    return o.view(q.shape)
