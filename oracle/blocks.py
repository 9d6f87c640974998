"""What stands around a checkpointed block, from its definitions, in fp64 numpy on
the CPU: activations in 8 bits, RMSNorm and its gradients, the norms after and
before a block, rotary positions.  The oracle of the GPU tests of these operators.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
MIN_EXP = -118


def _e4m3(v: np.ndarray) -> np.ndarray:
    """v rounded to e4m3 (ties to even, subnormals of 2^-9); |v| <= 448."""
    _, e = np.frexp(v)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(v / step) * step


def pack8(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """(code values [T, H] in fp64, exponent bytes [T, ceil(H / 32)]) of x [T, H]."""
    T, H = x.shape
    nb = -(-H // BLOCK)
    xb = np.zeros((T, nb * BLOCK))
    xb[:, :H] = x
    xb = xb.reshape(T, nb, BLOCK)
    bad = ~np.isfinite(xb).all(-1)
    xb = np.where(bad[..., None], 0.0, xb)
    m = np.abs(xb).max(-1)
    e = np.where(m > 0, np.frexp(m)[1] - 1, -1000)
    if fmt == "int8":
        E = np.maximum(e - 6, MIN_EXP)
        c = np.clip(np.rint(xb * np.ldexp(1.0, -E)[..., None]), -127, 127)
    else:
        E = np.maximum(e - 8, MIN_EXP)
        E = E + (m * np.ldexp(1.0, -E) > 448)
        c = _e4m3(xb * np.ldexp(1.0, -E)[..., None])
        c = np.where((E == 120)[..., None], np.clip(c, -240, 240), c)  # 256 * 2^120 is no finite fp32 or bf16
    return c.reshape(T, nb * BLOCK)[:, :H], np.where(bad, 255, E + 127).astype(np.uint8)


def unpack8(codes: np.ndarray, exps: np.ndarray) -> np.ndarray:
    scale = np.where(exps == 255, np.nan, np.ldexp(1.0, exps.astype(np.int64) - 127))
    return codes * np.repeat(scale, BLOCK, 1)[:, :codes.shape[1]]


def rmsnorm(x: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rmsnorm_bwd(dy: np.ndarray, x: np.ndarray, w: np.ndarray, eps: float):
    """(dx, dw, and what dx's roundings act on: r |dy w| + r |n| mean |dy w n|)."""
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, g = x * r, dy * w
    dx = r * (g - n * (g * n).mean(-1, keepdims=True))
    terms = r * (np.abs(g) + np.abs(n) * np.abs(g * n).mean(-1, keepdims=True))
    return dx, (dy * n).sum(0), terms


def block_norms(x, a, w_post, w_pre, gate, scale, eps, h=None):
    """(h, y or None); with h given (as stored), y is its norm."""
    n = a if w_post is None else rmsnorm(a, w_post, eps)
    s = x + scale * (1.0 if gate is None else gate) * n
    return s, None if w_pre is None else rmsnorm(s if h is None else h, w_pre, eps)


def block_norms_bwd(dh, dy, h, a, w_post, w_pre, gate, scale, eps):
    """{name: (gradient, what fp32 roundings act on)} of block_norms at the stored h: the
    second of each pair sums the magnitudes that its fp32 arithmetic adds up."""
    g = 1.0 if gate is None else gate
    D, mag, out = dh, np.abs(dh), {}
    if w_pre is not None:
        dn, _, terms = rmsnorm_bwd(dy, h, w_pre, eps)
        D, mag = D + dn, mag + terms
        n = rmsnorm(h, 1.0, eps)
        out["dw_pre"] = (dy * n).sum(0), np.abs(dy * n).sum(0)
    out["dx"] = D, mag
    P, pmag = scale * g * D, np.abs(scale * g) * mag
    n = a if w_post is None else rmsnorm(a, 1.0, eps)
    nw = n if w_post is None else n * w_post
    if w_post is not None:
        out["dw_post"] = (P * n).sum(0), (pmag * np.abs(n)).sum(0)
        out["da"] = rmsnorm_bwd(P, a, w_post, eps)[0], rmsnorm_bwd(pmag, np.abs(a), np.abs(w_post), eps)[2]
    else:
        out["da"] = P, pmag
    if gate is not None:
        dg, gmag = scale * D * nw, np.abs(scale * nw) * mag
        out["dgate"] = (dg, gmag) if gate.ndim > 1 else (dg.sum(0), gmag.sum(0))
    return out


def rotary(x, pos, inv_freq, head_dim, offset, layout, factor, back=False):
    """(x [T, heads * head_dim] turned, the magnitudes its roundings act on)."""
    T, n = x.shape[0], len(inv_freq)
    i = np.arange(n)
    u, v = (offset + i, offset + n + i) if layout == "half" else (offset + 2 * i, offset + 2 * i + 1)
    angle = np.resize(pos, T).astype(np.float64)[:, None] * inv_freq
    c, s = factor * np.cos(angle)[:, None], factor * np.sin(-angle if back else angle)[:, None]
    y = x.reshape(T, -1, head_dim).copy()
    mag = np.zeros_like(y)
    x0, x1 = y[..., u].copy(), y[..., v].copy()
    y[..., u], y[..., v] = x0 * c - x1 * s, x1 * c + x0 * s
    mag[..., u] = mag[..., v] = abs(factor) * (np.abs(x0) + np.abs(x1))
    return y.reshape(T, -1), mag.reshape(T, -1)
