"""Rotary positions from positions and frequencies: the half and the interleaved layout,
part of a head or all of it, frequencies scaled for long contexts.

The stock layer's rotation (transformers 5.15.0, models/llama/modeling_llama.py:130-160)
reads cos/sin tables in the model's dtype, laid out for every position by the model
(femtotron/model/llama_partial_model.py:196-203), and turns whole heads in the half layout
(``ops.rope_fwd_``).  Here the angles are computed where they are used, in fp64 up to the
turn's remainder, so far positions and packed sequences need no table.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import ops

SCALINGS = ("default", "linear", "dynamic", "yarn", "llama3")


def rotary_frequencies(rot_dim: int, theta: float | None = None, scaling: dict | None = None, *,
                       seq_len: int | None = None, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, factor) of ``apply_rotary``: the angle a position of each of the rot_dim / 2
    pairs (float64), theta^(-2i / rot_dim) unless scaled, and the factor on cos and sin.

    ``theta``: given here, or else ``scaling``'s "rope_theta" (two that differ are refused),
    or 10000.  ``rot_dim`` is what is rotated of a head: "partial_rotary_factor" is not read.

    ``scaling``: the dict of a Hugging Face config (``rope_scaling``), its "rope_type"
    (or "type") one of
      "default"  unscaled;
      "linear"   positions divided by "factor";
      "dynamic"  theta raised for a sequence of ``seq_len`` past
                 "original_max_position_embeddings" (NTK-aware), by "factor"; a config
                 has that length as its max_position_embeddings, to be put in;
      "yarn"     pairs that turn fewer than "beta_slow" times in the original context
                 divided by "factor", more than "beta_fast" times kept, a ramp between
                 (its ends at whole pairs unless "truncate" is False);
                 the factor on cos and sin is "attention_factor", or
                 0.1 "mscale" ln("factor") + 1 over the same of "mscale_all_dim";
      "llama3"   wavelengths over original / "low_freq_factor" divided by "factor", under
                 original / "high_freq_factor" kept, a ramp in the frequency between.
    """
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be positive and even, got {rot_dim}")
    scaling = dict(scaling or {})
    layers = [k for k, v in scaling.items() if isinstance(v, dict)]
    if layers:
        raise ValueError(f"scaling holds one dict for each of {layers}: pass the one of the layer")
    own = scaling.get("rope_theta")
    if theta is None:
        theta = 10000.0 if own is None else float(own)
    elif own is not None and float(own) != float(theta):
        raise ValueError(f"theta is {theta}, the scaling's rope_theta {own}")
    if not theta > 1:
        raise ValueError(f"theta must be over 1, got {theta}")
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in SCALINGS:
        raise ValueError(f"rope_type must be one of {SCALINGS}, got {kind!r}")

    def need(key):
        if scaling.get(key) is None:
            raise ValueError(f"{kind!r} scaling needs {key!r}")
        return float(scaling[key])

    theta = float(theta)
    n = rot_dim // 2
    pair = torch.arange(n, dtype=torch.float64)
    attention = 1.0
    if kind == "dynamic":
        original, by = need("original_max_position_embeddings"), need("factor")
        if rot_dim == 2:
            raise ValueError("'dynamic' scaling needs rot_dim over 2")
        length = max(float(seq_len or 0), original)
        theta *= (by * length / original - (by - 1)) ** (rot_dim / (rot_dim - 2))
    freq = theta ** (-pair / n)
    if kind == "linear":
        freq = freq / need("factor")
    elif kind == "llama3":
        original, by = need("original_max_position_embeddings"), need("factor")
        low, high = need("low_freq_factor"), need("high_freq_factor")
        if not high > low:
            raise ValueError("'llama3' scaling needs high_freq_factor over low_freq_factor")
        turns = original * freq / (2 * math.pi)  # in the original context
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / by)
    elif kind == "yarn":
        original, by = need("original_max_position_embeddings"), need("factor")
        fast, slow = (float(scaling.get(k) or d) for k, d in (("beta_fast", 32), ("beta_slow", 1)))
        # the (real) pair that turns b times in the original context
        at = [n * math.log(original / (2 * math.pi * b)) / math.log(theta) for b in (fast, slow)]
        if scaling.get("truncate", True):
            at = [math.floor(at[0]), math.ceil(at[1])]
        lo, hi = max(at[0], 0), min(at[1], rot_dim - 1)
        divide = ((pair - lo) / (hi - lo if hi != lo else 0.001)).clamp(0, 1)
        freq = freq * (1 - divide + divide / by)
        attention = scaling.get("attention_factor")
        if attention is None:
            def grown(m):
                return 0.1 * m * math.log(by) + 1.0 if by > 1 else 1.0
            m, all_dim = scaling.get("mscale"), scaling.get("mscale_all_dim")
            attention = grown(m) / grown(all_dim) if m and all_dim else grown(1.0)
    return freq.to(device), float(attention)


class RotaryFunction(torch.autograd.Function):
    """Saved: the positions and frequencies."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, how):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return _turn(ops.rotary_fwd, q, k, positions, inv_freq, how)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 5
        return (*_turn(ops.rotary_bwd, dq, dk, positions, inv_freq, ctx.how), None, None, None)


def _rows(t: torch.Tensor | None) -> torch.Tensor | None:
    """t as token rows: a view where it is one, laid out first where it is none (a
    transposed or an expanded gradient)."""
    if t is None:
        return None
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    ld, unit = t.stride()
    return t if unit == 1 and ld >= t.shape[1] else t.contiguous()


def _turn(op, q, k, positions, inv_freq, how):
    qo, ko = op(_rows(q), _rows(k), positions, inv_freq, **how)
    return (qo if q is None or q.dim() == 2 else qo.view(q.shape),
            ko if k is None or k.dim() == 2 else ko.view(k.shape))


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 head_dim: int, rot_dim: int | None = None, offset: int = 0, layout: str = "half",
                 factor: float = 1.0) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q and k, [tokens, heads * head_dim] or [batch, seq, heads * head_dim] (k may be None,
    their head counts may differ; column views of a packed projection are read in place),
    with dims [offset, offset + rot_dim) of each head turned by positions * inv_freq, cos
    and sin times factor; differentiable in q and k (once, and in reverse mode).

    positions: int64 of any shape, one a token in order, or one a position of sequences of
    equal length (seq of them; of [tokens, ...] a divisor of tokens); inv_freq, factor:
    ``rotary_frequencies``, constants (refused where they want a gradient); layout: pairs (i, i + rot_dim / 2), "half", or (2i, 2i + 1),
    "interleaved"."""
    if ops.wants_derivative(inv_freq) or ops.wants_derivative(factor):
        raise TypeError("apply_rotary: inv_freq and factor are constants and get no gradient")
    n_positions = positions.numel()
    for t, n in ((q, "q"), (k, "k")):
        if t is None:
            continue
        if t.dim() not in (2, 3):
            raise ValueError(f"apply_rotary: {n} must be [tokens, heads * head_dim] or [batch, seq, heads * head_dim] "
                             f"(heads and head_dim in one dim), got {tuple(t.shape)}")
        if t.dim() == 3 and n_positions not in (t.shape[1], t.shape[0] * t.shape[1]):
            raise ValueError(f"apply_rotary: {n_positions} positions are neither one a token nor one a position of "
                             f"{n} {tuple(t.shape)}")
    how = dict(head_dim=head_dim, rot_dim=rot_dim, offset=offset, layout=layout, factor=float(factor))
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    if ops.differentiated(q, k):
        return RotaryFunction.apply(q, k, positions, inv_freq, how)
    return _turn(ops.rotary_fwd, q, k, positions, inv_freq, how)
