"""Attention under a mask in fp64, from its definition, with bounds on what fp32 sums and the
kernels' roundings may leave: the oracle of the tests of masked and cached attention."""
from __future__ import annotations

import math

import torch


def ranges(batch, seq, starts=None, lengths=None, prefix=None, window=None, causal=True):
    """(lo, hi) lists: what each token sees, token by token (include/femtohip_packed.h)."""
    T = batch * seq
    if starts is None:
        starts = [b * seq for b in range(batch)]
        ends = [s + seq for s in starts]
    else:
        ends = list(starts[1:]) + [T]
    if lengths is not None:
        ends = [min(e, s + max(n, 0)) for s, e, n in zip(starts, ends, lengths)]
    lo, hi = [0] * T, [0] * T
    for d, (s, e) in enumerate(zip(starts, ends)):
        for t in range(s, min(e, T)):
            lo[t], hi[t] = s, t + 1 if causal else e
            if prefix is not None:
                hi[t] = max(t + 1, min(s + max(prefix[d], 0), e))
            if window is not None:
                lo[t] = max(s, t + 1 - window)
                hi[t] = min(hi[t], t + window)
    return lo, hi


def seen(lo, hi, n_keys, device):
    j = torch.arange(n_keys, device=device)
    lo, hi = (torch.tensor(x, device=device)[:, None] for x in (lo, hi))
    return (lo <= j) & (j < hi)


def heads(x, head_dim):
    """[rows, heads * head_dim] as [heads, rows, head_dim] in fp64."""
    return x.detach().double().unflatten(-1, (-1, head_dim)).transpose(0, 1)


def rows(x):
    return x.transpose(0, 1).flatten(1)


def attention(q, k, v, see, away, head_dim, *, scale=None, cap=None, slopes=None, do=None, dtype=None):
    """{"o", ...} and its bounds {"o", ...} for q [n, H D], k and v [m, Hk D], see [n, m] and
    distances away [n, m]; with do also dq, dk, dv.  dtype: the kernels'.

    The bounds count, with u = eps / 2 of the dtype, f = 2^-24 and n terms a sum: an output's
    rounding u; u on each weight (and each dS) that bf16 products take; a score's error e_s
    from sums of head_dim products and from what tanh, exp2 and the distances' products
    leave; n f on each sum; o's own error in delta (its weights' rounding and 2^-17 of its
    size, all of fp32's u of it in fp32)."""
    scale = head_dim ** -0.5 if scale is None else scale
    f = 2.0 ** -24
    u = torch.finfo(dtype).eps / 2
    uw = u if dtype == torch.bfloat16 else 0.0  # on the weights
    Q, K, V = heads(q, head_dim), heads(k, head_dim), heads(v, head_dim)
    group = Q.shape[0] // K.shape[0]
    Kq, Vq = K.repeat_interleave(group, 0), V.repeat_interleave(group, 0)
    s = scale * (Q @ Kq.mT)
    G = scale * (Q.abs() @ Kq.abs().mT)
    t = torch.zeros_like(s)
    z = s
    if cap:
        t = torch.tanh(s / cap)
        z = cap * t
    zb = z
    if slopes is not None:
        zb = z - slopes.double()[:, None, None] * away.abs()
    w = torch.softmax(zb.masked_fill(~see, -math.inf), -1)
    p = torch.where(see, w, 0.0)
    p = torch.where(see.any(-1)[:, None], p, 0.0)
    o = p @ Vq
    n = see.sum(-1).max().item() + head_dim
    # a score in log2 units, relative to the weight: products, z's roundings, the cap's tanh, exp2
    top = torch.where(see, zb.abs(), 0.0).amax(-1, keepdim=True)
    e_s = f * ((head_dim + 4) * torch.where(see, G, 0.0).amax(-1, keepdim=True) + 8 * top + 8 * (cap or 0.0) + 8)
    A = p @ Vq.abs()
    e_o = (uw + 2 * e_s + 2 * n * f) * (A + o.abs())  # before o's rounding
    out, tol = {"o": rows(o)}, {"o": rows(u * o.abs() + e_o) + 1e-30}
    if do is None:
        return out, tol
    dO = heads(do, head_dim)
    dp = dO @ Vq.mT
    delta = (dO * o).sum(-1, keepdim=True)
    slope = 1 - t.square()
    ds = p * (dp - delta) * slope
    e_delta = (dO.abs() * (e_o + (2.0 ** -17 if uw else u) * o.abs())).sum(-1, keepdim=True) \
        + head_dim * f * (dO.abs() * o.abs()).sum(-1, keepdim=True)
    e_dp = head_dim * f * (dO.abs() @ Vq.abs().mT)
    # e_lse is e_s's; the derivative of the cap is off by 8 f
    e_ds = (uw + 4 * e_s + 4 * n * f) * ds.abs() + p * slope * (e_delta + e_dp) + 8 * f * p * (dp - delta).abs()
    e_p = (uw + 4 * e_s + 2 * n * f) * p

    def per_kv(x):
        return x.unflatten(0, (-1, group)).sum(1)

    N = see.sum(0).max().item() * group + head_dim
    g = {"dq": scale * (ds @ Kq), "dk": per_kv(scale * (ds.mT @ Q)), "dv": per_kv(p.mT @ dO)}
    e = {"dq": scale * (e_ds @ Kq.abs() + n * f * (ds.abs() @ Kq.abs())),
         "dk": per_kv(scale * (e_ds.mT @ Q.abs() + N * f * (ds.abs().mT @ Q.abs()))),
         "dv": per_kv(e_p.mT @ dO.abs() + N * f * (p.mT @ dO.abs()))}
    for name in g:
        out[name] = rows(g[name])
        tol[name] = rows(u * g[name].abs() + e[name]) + 1e-30
    return out, tol


def check(got, want, tol, name=""):
    """Every element within its bound (finite), with the worst one named."""
    got = got.detach().double().reshape(want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - want).abs() / tol).max().item() if want.numel() else 0.0
    assert over <= 1.0, f"{name}: {over:.2f} times its bound"
