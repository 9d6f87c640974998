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
