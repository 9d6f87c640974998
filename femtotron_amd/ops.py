"""Torch-tensor front end of the femtohip C ABI.

Each function validates device, dtype, shape and strides on the host, then
calls the matching ``fh_*`` entry point on the tensor's current HIP stream.
Outputs are allocated by the caller or here with ``torch.empty`` (PyTorch's
caching allocator); the library itself never allocates device memory.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DT = {torch.bfloat16: _lib.FH_BF16, torch.float32: _lib.FH_F32}


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"femtohip supports bfloat16 and float32, got {t.dtype}") from None


def _require_gpu(*ts: torch.Tensor) -> None:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("femtohip ops take HIP device tensors only")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")


def _same_dtype(ref: torch.Tensor, *ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and t.dtype != ref.dtype:
            raise TypeError(f"dtype mismatch: {t.dtype} vs {ref.dtype}")


def _alike(ref: torch.Tensor, *ts: torch.Tensor | None) -> None:
    """Every tensor on ref's HIP device and of its dtype (_require_gpu and _same_dtype in one pass)."""
    dev, dt = ref.get_device(), ref.dtype
    if dev < 0:
        raise ValueError("femtohip ops take HIP device tensors only")
    for t in ts:
        if t is None:
            continue
        if t.get_device() != dev:
            _require_gpu(ref, t)
        if t.dtype != dt:
            raise TypeError(f"dtype mismatch: {t.dtype} vs {dt}")


def _row_stats(name: str, like: torch.Tensor, rows: int, *rs: torch.Tensor | None) -> None:
    """Per-row fp32 statistics (rstd): on like's device, contiguous, one entry a row."""
    for r in rs:
        if r is None:
            continue
        if r.get_device() != like.get_device():
            _require_gpu(like, r)
        if r.dtype != torch.float32 or r.numel() != rows or not r.is_contiguous():
            raise ValueError(f"{name}: rstd must be contiguous fp32 with one entry per row")


def _rowmajor(t: torch.Tensor, name: str) -> int:
    """Row stride of a 2-D view whose last dim is contiguous."""
    if t.dim() != 2 or (t.size(1) > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: expected a 2-D view with a contiguous last dim, got "
                         f"shape {tuple(t.shape)} strides {t.stride()}")
    return t.stride(0)


def _stream(t: torch.Tensor) -> int:
    """The current stream of t's device (the raw handle: building a
    torch.cuda.Stream object costs more than the launch's other host work)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_jit_trace, _mode = torch._C._get_tracing_state, torch._C._get_dispatch_mode
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _launch(name: str, t: torch.Tensor, *args) -> None:
    """Calls an entry point on the current stream of t's device, with that device
    the current one (the default stream's handle is 0 on every device).  Refused while
    torch records the operations it sees, of which a kernel is none."""
    if _jit_trace() is not None or _mode(_PROXY) is not None:
        raise RuntimeError(f"{name}: torch.jit.trace and make_fx do not see this library's kernels; "
                           "a trace would return uninitialised memory")
    index = t.get_device()
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
        return
    status = getattr(_lib.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def aligned(t: torch.Tensor | None) -> torch.Tensor | None:
    """t contiguous and 16-byte aligned, as the kernels take it: itself, or a copy."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def differentiated(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these tensors has to go through its autograd node: one wants a
    gradient, or forward-mode derivatives are on (their dual tensors do not say that they
    want one, and the node is what refuses them: it has no jvp)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0


def wants_derivative(v) -> bool:
    """Whether v, a constant of an operator, is a tensor that asks for a derivative."""
    return isinstance(v, torch.Tensor) and ((v.requires_grad and torch.is_grad_enabled())
                                            or (forward_ad._current_level >= 0
                                                and forward_ad.unpack_dual(v).tangent is not None))


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _fptr(t: torch.Tensor | None):
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise TypeError("fp32 tensor expected")
    return ctypes.cast(t.data_ptr(), ctypes.POINTER(ctypes.c_float))


# ------------------------------------------------------------------ RMSNorm
def rmsnorm_fwd(x: torch.Tensor, w: torch.Tensor, eps: float, *, out: torch.Tensor | None = None,
                rstd: torch.Tensor | None = None) -> torch.Tensor:
    """y = w * to_dtype(x * rsqrt(mean(x^2) + eps)) over the last dim of contiguous x."""
    _require_gpu(x, w, out, rstd)
    _same_dtype(x, w, out)
    if not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("rmsnorm_fwd: x and w must be contiguous")
    cols = x.size(-1)
    rows = x.numel() // max(cols, 1)
    if w.numel() != cols:
        raise ValueError("rmsnorm_fwd: weight size != last dim")
    y = torch.empty_like(x) if out is None else out
    if rstd is not None and rstd.numel() != rows:
        raise ValueError("rmsnorm_fwd: rstd must have one entry per row")
    _lib.call("fh_rmsnorm_fwd", _dtype_code(x), _ptr(x), _ptr(w), _ptr(y), _fptr(rstd), rows,
              cols, float(eps), _stream(x))
    return y


def add_rmsnorm_fwd(x: torch.Tensor, a: torch.Tensor, w: torch.Tensor, eps: float, *,
                    rstd: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """h = to_dtype(x + a); y = rmsnorm(h). Returns (h, y)."""
    _require_gpu(x, a, w, rstd)
    _same_dtype(x, a, w)
    if not (x.is_contiguous() and a.is_contiguous() and w.is_contiguous()):
        raise ValueError("add_rmsnorm_fwd: inputs must be contiguous")
    if x.shape != a.shape:
        raise ValueError("add_rmsnorm_fwd: x and a shapes differ")
    cols = x.size(-1)
    rows = x.numel() // max(cols, 1)
    if w.numel() != cols:
        raise ValueError("add_rmsnorm_fwd: weight size != last dim")
    h = torch.empty_like(x)
    y = torch.empty_like(x)
    _lib.call("fh_add_rmsnorm_fwd", _dtype_code(x), _ptr(x), _ptr(a), _ptr(w), _ptr(h), _ptr(y),
              _fptr(rstd), rows, cols, float(eps), _stream(x))
    return h, y


def rmsnorm_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, eps: float, *,
                rstd: torch.Tensor | None = None, dres: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of rmsnorm_fwd: returns (dx [+ dres], dw)."""
    _require_gpu(dy, x, w, rstd, dres)
    _same_dtype(x, dy, w, dres)
    for t, n in ((dy, "dy"), (x, "x"), (w, "w"), (dres, "dres")):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"rmsnorm_bwd: {n} must be contiguous")
    if dy.shape != x.shape or (dres is not None and dres.shape != x.shape):
        raise ValueError("rmsnorm_bwd: shape mismatch")
    cols = x.size(-1)
    rows = x.numel() // max(cols, 1)
    if w.numel() != cols:
        raise ValueError("rmsnorm_bwd: weight size != last dim")
    dx = torch.empty_like(x)
    dw = torch.empty_like(w)
    ws_bytes = _lib.lib().fh_rmsnorm_bwd_workspace_size(rows, cols)
    ws = torch.empty(max(ws_bytes, 4) // 4, dtype=torch.float32, device=x.device)
    _lib.call("fh_rmsnorm_bwd", _dtype_code(x), _ptr(dy), _ptr(x), _ptr(w), _fptr(rstd),
              _ptr(dres), _ptr(dx), _ptr(dw), _ptr(ws), rows, cols, float(eps), _stream(x))
    return dx, dw


# ------------------------------------------------------- activations in 8 bits
class Packed8(NamedTuple):
    """An activation kept in 8 bits (include/femtohip_blocks.h): codes, int8 or
    float8_e4m3fn of the activation's shape, and the exponent bytes, uint8 [...,
    ceil(cols / 32)], of its blocks of 32 elements."""
    codes: torch.Tensor
    exps: torch.Tensor


_FMT8 = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FORMATS8 = tuple(_FMT8)
_FMT8_CODE = {torch.int8: _lib.FH_INT8, torch.float8_e4m3fn: _lib.FH_E4M3}


def _empty8(x: torch.Tensor, fmt: str) -> Packed8:
    if fmt not in _FMT8:
        raise ValueError(f"8-bit format must be one of {FORMATS8}, got {fmt!r}")
    if x.dim() == 0 or x.size(-1) % 8:
        raise ValueError(f"an activation's last dim must be a multiple of 8 to be packed, got shape {tuple(x.shape)}")
    return Packed8(torch.empty_like(x, dtype=_FMT8[fmt]), x.new_empty((*x.shape[:-1], -(-x.size(-1) // 32)), dtype=torch.uint8))


def _packed(name: str, p: Packed8) -> tuple[int, int, int]:
    """(format code, rows, cols) of a packed activation, checked."""
    codes, exps = p
    fmt = _FMT8_CODE.get(codes.dtype)
    if fmt is None or exps.dtype != torch.uint8:
        raise TypeError(f"{name}: codes must be int8 or float8_e4m3fn and exps uint8, got {codes.dtype}, {exps.dtype}")
    if codes.get_device() < 0 or codes.get_device() != exps.get_device():
        _require_gpu(codes, exps)
    shape = codes.shape
    if not shape or not codes.is_contiguous() or not exps.is_contiguous():
        raise ValueError(f"{name}: codes and exps must be contiguous")
    cols = shape[-1]
    if exps.shape != (*shape[:-1], -(-cols // 32)):
        raise ValueError(f"{name}: exps {tuple(exps.shape)} are not those of codes {tuple(shape)}")
    return fmt, codes.numel() // max(cols, 1), cols


def pack8(x: torch.Tensor, fmt: str = "int8") -> Packed8:
    """A contiguous x in 8.25 bits an element: blocks of 32 along the last dim with one
    power-of-two exponent, codes "int8" or "e4m3" (fh_pack8)."""
    _alike(x)
    dt = _dtype_code(x)
    if not x.is_contiguous():
        raise ValueError("pack8: x must be contiguous")
    codes, exps = p = _empty8(x, fmt)
    cols = x.size(-1)
    if x.numel():
        _launch("fh_pack8", x, dt, _FMT8_CODE[codes.dtype], _ptr(x), _ptr(codes), _ptr(exps), x.numel() // cols, cols)
    return p


def unpack8(p: Packed8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values a packed activation stands for; bf16 and fp32 hold them exactly (fh_unpack8)."""
    fmt, rows, cols = _packed("unpack8", p)
    x = torch.empty_like(p.codes, dtype=dtype)
    dt = _dtype_code(x)
    if x.numel():
        _launch("fh_unpack8", x, dt, fmt, _ptr(p.codes), _ptr(p.exps), _ptr(x), rows, cols)
    return x


def _norm8_args(name: str, codes: torch.Tensor, w: torch.Tensor, cols: int, rows: int, rstd: torch.Tensor | None) -> int:
    """The dtype code of w, checked to be the weight of a norm over the rows of codes."""
    if w.get_device() != codes.get_device():
        _require_gpu(codes, w)
    if w.numel() != cols or not w.is_contiguous():
        raise ValueError(f"{name}: w must be contiguous, of the last dim's size")
    if rstd is not None:
        _row_stats(name, w, rows, rstd)
    return _dtype_code(w)


def rmsnorm_fwd_pack8(x: torch.Tensor, w: torch.Tensor, eps: float, fmt: str = "int8", *,
                      rstd: torch.Tensor | None = None, llama_rounding: bool = False) -> tuple[torch.Tensor, Packed8]:
    """RMSNorm of x, and pack8(x, fmt), in one pass over x.  Rounded once; with
    llama_rounding as rmsnorm_fwd is, the normalised value before its product with w."""
    _alike(x, w)
    if not x.is_contiguous():
        raise ValueError("rmsnorm_fwd_pack8: x must be contiguous")
    codes, exps = p = _empty8(x, fmt)
    cols = x.size(-1)
    rows = x.numel() // max(cols, 1)
    dt = _norm8_args("rmsnorm_fwd_pack8", x, w, cols, rows, rstd)
    y = torch.empty_like(x)
    _launch("fh_rmsnorm_fwd_pack8", x, dt, _FMT8_CODE[codes.dtype], _ptr(x), _ptr(w), _ptr(y), _ptr(codes), _ptr(exps),
            _ptr(rstd), rows, cols, eps, llama_rounding)
    return y, p


def rmsnorm_fwd8(p: Packed8, w: torch.Tensor, eps: float, *, rstd: torch.Tensor | None = None,
                 llama_rounding: bool = False) -> torch.Tensor:
    """RMSNorm of the packed x, in w's dtype; with llama_rounding the bits of
    rmsnorm_fwd(unpack8(p), w, eps)."""
    fmt, rows, cols = _packed("rmsnorm_fwd8", p)
    dt = _norm8_args("rmsnorm_fwd8", p.codes, w, cols, rows, rstd)
    y = torch.empty_like(p.codes, dtype=w.dtype)
    _launch("fh_rmsnorm_fwd8", w, dt, fmt, _ptr(p.codes), _ptr(p.exps), _ptr(w), _ptr(y), _ptr(rstd), rows, cols, eps,
            llama_rounding)
    return y


def add_rmsnorm_fwd8(p: Packed8, a: torch.Tensor, w: torch.Tensor, eps: float, *, rstd: torch.Tensor | None = None,
                     llama_rounding: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """h = to_dtype(x + a) of the packed x, and y = RMSNorm(h); with llama_rounding the bits
    of add_rmsnorm_fwd.  Returns (h, y)."""
    fmt, rows, cols = _packed("add_rmsnorm_fwd8", p)
    _alike(a, w)
    if a.shape != p.codes.shape or not a.is_contiguous():
        raise ValueError("add_rmsnorm_fwd8: a must be contiguous, of the packed x's shape")
    dt = _norm8_args("add_rmsnorm_fwd8", p.codes, w, cols, rows, rstd)
    h, y = torch.empty_like(a), torch.empty_like(a)
    _launch("fh_add_rmsnorm_fwd8", a, dt, fmt, _ptr(p.codes), _ptr(p.exps), _ptr(a), _ptr(w), _ptr(h), _ptr(y),
            _ptr(rstd), rows, cols, eps, llama_rounding)
    return h, y


def rmsnorm_bwd8(dy: torch.Tensor, p: Packed8, w: torch.Tensor, eps: float, *, rstd: torch.Tensor | None = None,
                 dres: torch.Tensor | None = None, llama_rounding: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of RMSNorm at the packed x: (dx [+ dres], dw); with llama_rounding the bits
    of rmsnorm_bwd."""
    fmt, rows, cols = _packed("rmsnorm_bwd8", p)
    _alike(dy, w, dres)
    for t, n in ((dy, "dy"), (dres, "dres")):
        if t is not None and (t.shape != p.codes.shape or not t.is_contiguous()):
            raise ValueError(f"rmsnorm_bwd8: {n} must be contiguous, of the packed x's shape")
    dt = _norm8_args("rmsnorm_bwd8", p.codes, w, cols, rows, rstd)
    dx, dw = torch.empty_like(dy), torch.empty_like(w)
    nbytes = _lib.lib().fh_rmsnorm_bwd8_workspace_size(rows, cols)
    ws = dy.new_empty(max(nbytes, 4), dtype=torch.uint8)
    _launch("fh_rmsnorm_bwd8", dy, dt, fmt, _ptr(dy), _ptr(p.codes), _ptr(p.exps), _ptr(w), _ptr(rstd), _ptr(dres),
            _ptr(dx), _ptr(dw), _ptr(ws), rows, cols, eps, llama_rounding)
    return dx, dw


# --------------------------------------------------------------------- RoPE
def _rope(name: str, qk: torch.Tensor, n_heads: int, head_dim: int, seq_len: int,
          cos: torch.Tensor, sin: torch.Tensor) -> None:
    _require_gpu(qk, cos, sin)
    _same_dtype(qk, cos, sin)
    ld = _rowmajor(qk, name)
    if qk.size(1) < n_heads * head_dim:
        raise ValueError(f"{name}: buffer narrower than n_heads*head_dim")
    tokens = qk.size(0)
    cos2, sin2, per_token = _rope_tables(name, cos, sin, head_dim, seq_len, tokens)
    _lib.call(name, _dtype_code(qk), _ptr(qk), ld, tokens, seq_len, n_heads, head_dim, _ptr(cos2),
              _ptr(sin2), per_token, _stream(qk))


def _rope_tables(name: str, cos: torch.Tensor, sin: torch.Tensor, head_dim: int, seq_len: int,
                 tokens: int):
    """cos/sin as [rows, head_dim] views and the cos_per_token flag of the C ABI:
    rows == seq_len (one row per position) or rows == tokens (one per token)."""
    cos2 = cos.reshape(-1, head_dim)
    sin2 = sin.reshape(-1, head_dim)
    if not (cos2.is_contiguous() and sin2.is_contiguous()) or cos2.shape != sin2.shape:
        raise ValueError(f"{name}: cos/sin must be contiguous and of equal shape")
    if cos2.size(0) == seq_len:
        if tokens % seq_len:
            raise ValueError(f"{name}: tokens not a multiple of seq_len")
        return cos2, sin2, 0
    if cos2.size(0) == tokens:
        return cos2, sin2, 1
    raise ValueError(f"{name}: cos/sin rows ({cos2.size(0)}) match neither seq_len nor tokens")


def rope_fwd_(qk: torch.Tensor, n_heads: int, head_dim: int, seq_len: int, cos: torch.Tensor,
              sin: torch.Tensor) -> torch.Tensor:
    """Rotate heads 0..n_heads-1 of the [tokens, ld] view qk in place."""
    _rope("fh_rope_fwd", qk, n_heads, head_dim, seq_len, cos, sin)
    return qk


def rope_bwd_(dqk: torch.Tensor, n_heads: int, head_dim: int, seq_len: int, cos: torch.Tensor,
              sin: torch.Tensor) -> torch.Tensor:
    _rope("fh_rope_bwd", dqk, n_heads, head_dim, seq_len, cos, sin)
    return dqk


# --------------------------------------------------- norms around a block
def _block_norms_shapes(name: str, like: torch.Tensor, w_post, w_pre, gate) -> tuple[int, int, int, int]:
    """(dtype code, gate_per_token, rows, cols) of block norms over `like`'s rows, checked."""
    shape = like.shape
    cols = shape[-1] if shape else 0
    if w_post is None and w_pre is None:
        raise ValueError(f"{name}: at least one of w_post and w_pre is needed")
    for w, n in ((w_post, "w_post"), (w_pre, "w_pre")):
        if w is not None and (w.shape != (cols,) or not w.is_contiguous()):
            raise ValueError(f"{name}: {n} must be a contiguous [{cols}] tensor, got {tuple(w.shape)}")
    per_token = 0
    if gate is not None:
        per_token = int(gate.shape != (cols,))
        if (per_token and gate.shape != shape) or not gate.is_contiguous():
            raise ValueError(f"{name}: gate must be contiguous, of shape [{cols}] or {tuple(shape)}, got "
                             f"{tuple(gate.shape)}")
    return _dtype_code(like), per_token, like.numel() // max(cols, 1), cols


def block_norms_check(name: str, x, a, w_post, w_pre, gate) -> tuple[int, int, int, int]:
    """_block_norms_shapes of the forward's tensors, all of which are checked."""
    _alike(x, a, w_post, w_pre, gate)
    args = _block_norms_shapes(name, x, w_post, w_pre, gate)
    if not x.is_contiguous() or not a.is_contiguous() or a.shape != x.shape:
        raise ValueError(f"{name}: x and a must be contiguous, of one shape")
    return args


def block_norms_fwd(x: torch.Tensor, a: torch.Tensor, w_post: torch.Tensor | None, w_pre: torch.Tensor | None, eps: float,
                    *, gate: torch.Tensor | None = None, scale: float = 1.0, rstd_post: torch.Tensor | None = None,
                    rstd_pre: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """h = to_dtype(x + scale * gate * rmsnorm(a; w_post)) and y = rmsnorm(h; w_pre), in
    fp32 between those roundings (fh_block_norms_fwd).  w_post None: a enters as it is;
    w_pre None: no y; gate [cols], of x's shape, or None.  Returns (h, y or None);
    rstd_post and rstd_pre (fp32, one a row) receive what block_norms_bwd reads."""
    args = block_norms_check("block_norms_fwd", x, a, w_post, w_pre, gate)
    _row_stats("block_norms_fwd", x, args[2], rstd_post, rstd_pre)
    return block_norms_fwd_checked(args, x, a, w_post, w_pre, gate, scale, eps, rstd_post, rstd_pre)


def block_norms_fwd_checked(args: tuple, x, a, w_post, w_pre, gate, scale, eps, rstd_post, rstd_pre):
    """block_norms_fwd of tensors that are known to fit; args: block_norms_check's."""
    dt, per_token, rows, cols = args
    h = torch.empty_like(x)
    y = None if w_pre is None else torch.empty_like(x)
    _launch("fh_block_norms_fwd", x, dt, _ptr(x), _ptr(a), _ptr(w_post), _ptr(w_pre), _ptr(gate), per_token, scale, _ptr(h),
            _ptr(y), _ptr(rstd_post), _ptr(rstd_pre), rows, cols, eps)
    return h, y


def block_norms_bwd(dh: torch.Tensor, dy: torch.Tensor | None, h: torch.Tensor | None, a: torch.Tensor | None,
                    w_post: torch.Tensor | None, w_pre: torch.Tensor | None, *, gate: torch.Tensor | None = None,
                    scale: float = 1.0, rstd_post: torch.Tensor | None = None, rstd_pre: torch.Tensor | None = None):
    """Gradients of block_norms_fwd: (dx, da, dw_post, dw_pre, dgate), None for what it
    did not have.  dy, h and rstd_pre go with w_pre, rstd_post with w_post, a with
    w_post or a gate."""
    _alike(dh, dy, h, a, w_post, w_pre, gate)
    args = _block_norms_shapes("block_norms_bwd", dh, w_post, w_pre, gate)
    if w_pre is not None and (dy is None or h is None or rstd_pre is None):
        raise ValueError("block_norms_bwd: w_pre needs dy, h and rstd_pre")
    if w_post is not None and rstd_post is None:
        raise ValueError("block_norms_bwd: w_post needs rstd_post")
    if a is None and (w_post is not None or gate is not None):
        raise ValueError("block_norms_bwd: w_post and a gate need a")
    for t, n in ((dh, "dh"), (dy, "dy"), (h, "h"), (a, "a")):
        if t is not None and (not t.is_contiguous() or t.shape != dh.shape):
            raise ValueError(f"block_norms_bwd: {n} must be contiguous, of dh's shape")
    _row_stats("block_norms_bwd", dh, args[2], rstd_post, rstd_pre)
    return block_norms_bwd_checked(args, dh, dy, h, a, w_post, w_pre, gate, scale, rstd_post, rstd_pre)


def block_norms_bwd_checked(args: tuple, dh, dy, h, a, w_post, w_pre, gate, scale, rstd_post, rstd_pre):
    """block_norms_bwd of tensors that are known to fit; args: block_norms_check's."""
    dt, per_token, rows, cols = args
    dx, da = torch.empty_like(dh), torch.empty_like(dh)
    dw_post, dw_pre, dgate = (None if t is None else torch.empty_like(t) for t in (w_post, w_pre, gate))
    nbytes = _lib.lib().fh_block_norms_bwd_workspace_size(rows, cols)
    ws = dh.new_empty(max(nbytes, 4), dtype=torch.uint8)
    _launch("fh_block_norms_bwd", dh, dt, _ptr(dh), _ptr(dy), _ptr(h), _ptr(a), _ptr(w_post), _ptr(w_pre), _ptr(gate),
            per_token, scale, _ptr(rstd_post), _ptr(rstd_pre), _ptr(dx), _ptr(da), _ptr(dw_post), _ptr(dw_pre),
            _ptr(dgate), _ptr(ws), rows, cols)
    return dx, da, dw_post, dw_pre, dgate


# ------------------------------------------------------- rotary positions
_ROTARY_LAYOUTS = {"half": _lib.FH_ROTARY_HALF, "interleaved": _lib.FH_ROTARY_INTERLEAVED}


def _rotary_rows(name: str, t: torch.Tensor, T: int, head_dim: int) -> int:
    """The row stride of a [T, heads * head_dim] view (of one row, which has none, its width)."""
    ld, shape = _rowmajor(t, name), t.shape
    if shape[0] != T or shape[1] % head_dim:
        raise ValueError(f"{name} must be [{T}, heads * {head_dim}], got {tuple(shape)}")
    return ld if T > 1 else shape[1]


def _rotary(name: str, q, k, positions: torch.Tensor, inv_freq: torch.Tensor, head_dim: int, rot_dim: int | None,
            offset: int, layout: str, factor: float, out):
    first = q if q is not None else k
    if first is None:
        raise ValueError(f"{name}: one of q and k is needed")
    qo, ko = (None, None) if out is None else out
    _alike(first, q, k, qo, ko)
    if positions.get_device() != first.get_device() or inv_freq.get_device() != first.get_device():
        _require_gpu(first, positions, inv_freq)
    dt, T = _dtype_code(first), first.size(0)
    if layout not in _ROTARY_LAYOUTS:
        raise ValueError(f"{name}: layout must be one of {tuple(_ROTARY_LAYOUTS)}, got {layout!r}")
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        raise TypeError(f"{name}: inv_freq must be contiguous float64")
    rot = 2 * inv_freq.numel() if rot_dim is None else rot_dim
    if inv_freq.dim() != 1 or rot != 2 * inv_freq.numel():
        raise ValueError(f"{name}: inv_freq must hold rot_dim / 2 values, got {tuple(inv_freq.shape)} for {rot}")
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        raise TypeError(f"{name}: positions must be contiguous int64")
    args = []
    outs = []
    for t, o, n in ((q, qo, "q"), (k, ko, "k")):
        if t is None:
            if o is not None:
                raise ValueError(f"{name}: an output for {n} without {n}")
            args.append((None, 0, 0, None, 0))
        else:
            ld = _rotary_rows(f"{name}: {n}", t, T, head_dim)
            if o is None:
                o = torch.empty_like(t, memory_format=torch.contiguous_format)
                lo = t.shape[1]
            elif o.shape != t.shape:
                raise ValueError(f"{name}: {n}'s output must have its shape")
            else:
                lo = _rotary_rows(f"{name}: {n}'s output", o, T, head_dim)
            args.append((t.data_ptr(), ld, t.shape[1] // head_dim, o.data_ptr(), lo))
        outs.append(o)
    n_positions = positions.numel()
    if T and (n_positions == 0 or T % n_positions):
        raise ValueError(f"{name}: {T} tokens are no multiple of {n_positions} positions")
    (qp, ldq, nq, qop, ldqo), (kp, ldk, nk, kop, ldko) = args
    _launch(name, first, dt, qp, ldq, nq, kp, ldk, nk, qop, ldqo, kop, ldko, T, head_dim, rot, offset,
            _ROTARY_LAYOUTS[layout], positions.data_ptr(), n_positions, inv_freq.data_ptr(), factor)
    return tuple(outs)


def rotary_fwd(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
               head_dim: int, rot_dim: int | None = None, offset: int = 0, layout: str = "half", factor: float = 1.0,
               out: tuple | None = None) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Turns the heads of the token-major views q and k [T, heads * head_dim] (either may
    be None) by positions * inv_freq in dims [offset, offset + rot_dim) of each head,
    pairs in the "half" or "interleaved" layout, cos and sin times factor; the other
    dims pass (fh_rotary_fwd).  positions: int64, one a token or one a position of
    sequences of equal length; inv_freq: float64 [rot_dim / 2].  `out`: (q, k) to
    write to, which may be the inputs.  Returns (q, k)."""
    return _rotary("fh_rotary_fwd", q, k, positions, inv_freq, head_dim, rot_dim, offset, layout, factor, out)


def rotary_bwd(dq: torch.Tensor | None, dk: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
               head_dim: int, rot_dim: int | None = None, offset: int = 0, layout: str = "half", factor: float = 1.0,
               out: tuple | None = None) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of rotary_fwd's inputs from those of its outputs: the turn back."""
    return _rotary("fh_rotary_bwd", dq, dk, positions, inv_freq, head_dim, rot_dim, offset, layout, factor, out)


# ------------------------------------------------------------------- SwiGLU
def swiglu_fwd(g: torch.Tensor, u: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """p = to_dtype(to_dtype(silu(g)) * u) for 2-D row-major views g, u (same row stride)."""
    _require_gpu(g, u, out)
    _same_dtype(g, u, out)
    ld_gu = _rowmajor(g, "swiglu_fwd.g")
    if _rowmajor(u, "swiglu_fwd.u") != ld_gu or g.shape != u.shape:
        raise ValueError("swiglu_fwd: g and u must share shape and row stride")
    rows, cols = g.shape
    p = torch.empty(rows, cols, dtype=g.dtype, device=g.device) if out is None else out
    _lib.call("fh_swiglu_fwd", _dtype_code(g), _ptr(g), _ptr(u), ld_gu, _ptr(p),
              _rowmajor(p, "swiglu_fwd.p"), rows, cols, _stream(g))
    return p


def swiglu_bwd(dp: torch.Tensor, g: torch.Tensor, u: torch.Tensor, dg: torch.Tensor,
               du: torch.Tensor, *, p_out: torch.Tensor | None = None) -> None:
    """dg, du of p = to_dtype(to_dtype(silu(g)) * u); with p_out, also writes p there (bit for
    bit swiglu_fwd's result).  p_out may be dp itself, which is then overwritten."""
    _require_gpu(dp, g, u, dg, du, p_out)
    _same_dtype(g, dp, u, dg, du, p_out)
    ld_gu = _rowmajor(g, "swiglu_bwd.g")
    ld_d = _rowmajor(dg, "swiglu_bwd.dg")
    if _rowmajor(u, "swiglu_bwd.u") != ld_gu or _rowmajor(du, "swiglu_bwd.du") != ld_d:
        raise ValueError("swiglu_bwd: g/u and dg/du must share row strides")
    if not (dp.shape == g.shape == u.shape == dg.shape == du.shape):
        raise ValueError("swiglu_bwd: shape mismatch")
    if p_out is not None and p_out.shape != g.shape:
        raise ValueError("swiglu_bwd: p_out shape mismatch")
    rows, cols = g.shape
    ld_p = _rowmajor(p_out, "swiglu_bwd.p_out") if p_out is not None else 0
    _lib.call("fh_swiglu_bwd", _dtype_code(g), _ptr(dp), _rowmajor(dp, "swiglu_bwd.dp"), _ptr(g),
              _ptr(u), ld_gu, _ptr(dg), _ptr(du), ld_d, _ptr(p_out), ld_p,
              rows, cols, _stream(g))


def scale(x: torch.Tensor, s: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """to_dtype(x * s) (fh_scale) for a contiguous bf16/fp32 x and an fp32 scalar tensor s on the
    same device; what ``(x * s).to(x.dtype)`` gives, in one streaming pass."""
    _require_gpu(x, s, out)
    if not x.is_contiguous() or s.numel() != 1 or s.dtype != torch.float32:
        raise ValueError("scale: x must be contiguous and s a one-element fp32 tensor")
    o = torch.empty_like(x) if out is None else out
    _same_dtype(x, o)
    if o.shape != x.shape or not o.is_contiguous():
        raise ValueError("scale: out must be a contiguous tensor of x's shape")
    sc = s.contiguous()
    _lib.call("fh_scale", _dtype_code(x), _ptr(x), _ptr(o), x.numel(), _ptr(sc), _stream(x))
    return o


def add(a: torch.Tensor, b: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_gpu(a, b, out)
    _same_dtype(a, b, out)
    if not (a.is_contiguous() and b.is_contiguous()) or a.shape != b.shape:
        raise ValueError("add: a and b must be contiguous with equal shapes")
    o = torch.empty_like(a) if out is None else out
    _lib.call("fh_add", _dtype_code(a), _ptr(a), _ptr(b), _ptr(o), a.numel(), _stream(a))
    return o


# ---------------------------------------------------------------- attention
def attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: int, seq_len: int,
             n_heads: int, n_kv_heads: int, head_dim: int, scale: float, *,
             need_lse: bool = True, rope: tuple | None = None,
             q_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Causal GQA attention on token-major [T, *] views (head h at columns h*head_dim).
    Returns (o [T, n_heads*head_dim], lse fp32 [batch, n_heads, seq_len] or None).
    rope=(cos, sin): q is read unrotated and rotated on load (fh_attn_fwd_rope; k
    must already be rotated); q_out (may be q itself) then receives the rotated q."""
    _require_gpu(q, k, v, q_out)
    _same_dtype(q, k, v)
    T = batch * seq_len
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        if t.size(0) != T:
            raise ValueError(f"attn_fwd: {n} has {t.size(0)} rows, expected {T}")
    o = torch.empty(T, n_heads * head_dim, dtype=q.dtype, device=q.device)
    lse = (torch.empty(batch, n_heads, seq_len, dtype=torch.float32, device=q.device)
           if need_lse else None)
    head = (_dtype_code(q), _ptr(q), _rowmajor(q, "q"), _ptr(k), _rowmajor(k, "k"),
            _ptr(v), _rowmajor(v, "v"), _ptr(o), o.stride(0), _fptr(lse))
    tail = (batch, seq_len, n_heads, n_kv_heads, head_dim, float(scale))
    if rope is None:
        if q_out is not None:
            raise ValueError("attn_fwd: q_out needs rope")
        _lib.call("fh_attn_fwd", *head, *tail, _stream(q))
        return o, lse
    cos, sin = rope
    _require_gpu(cos, sin)
    _same_dtype(q, cos, sin)
    if q_out is not None:
        _same_dtype(q, q_out)
        if tuple(q_out.shape) != tuple(q.shape):
            raise ValueError("attn_fwd: q_out must have q's shape")
    cos2, sin2, per_token = _rope_tables("attn_fwd_rope", cos, sin, head_dim, seq_len, T)
    _lib.call("fh_attn_fwd_rope", *head, _ptr(q_out), 0 if q_out is None else _rowmajor(q_out, "q_out"),
              *tail, _ptr(cos2), _ptr(sin2), per_token, _stream(q))
    return o, lse


def attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
             dout: torch.Tensor, lse: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor,
             dv: torch.Tensor, batch: int, seq_len: int, n_heads: int, n_kv_heads: int,
             head_dim: int, scale: float, rope: tuple | None = None) -> None:
    """Writes dq, dk, dv (token-major views, may be column ranges of one buffer).
    rope=(cos, sin): dq and dk come out passed through the RoPE backward as well
    (fh_attn_bwd_rope), the gradients before the rotation of q and k."""
    _require_gpu(q, k, v, o, dout, lse, dq, dk, dv)
    _same_dtype(q, k, v, o, dout, dq, dk, dv)
    if lse.dtype != torch.float32 or not lse.is_contiguous() or lse.numel() != batch * n_heads * seq_len:
        raise ValueError("attn_bwd: lse must be contiguous fp32 [batch, n_heads, seq_len]")
    ws_bytes = _lib.lib().fh_attn_bwd_call_workspace_size(_dtype_code(q), batch, seq_len, n_heads, n_kv_heads, head_dim)
    ws = torch.empty(max(ws_bytes, 4) // 4, dtype=torch.float32, device=q.device)
    args = (_dtype_code(q), _ptr(q), _rowmajor(q, "q"), _ptr(k), _rowmajor(k, "k"),
            _ptr(v), _rowmajor(v, "v"), _ptr(o), _rowmajor(o, "o"), _ptr(dout),
            _rowmajor(dout, "dout"), _fptr(lse), _ptr(dq), _rowmajor(dq, "dq"), _ptr(dk),
            _rowmajor(dk, "dk"), _ptr(dv), _rowmajor(dv, "dv"), _ptr(ws), batch, seq_len,
            n_heads, n_kv_heads, head_dim, float(scale))
    if rope is None:
        _lib.call("fh_attn_bwd", *args, _stream(q))
        return
    cos, sin = rope
    _require_gpu(cos, sin)
    _same_dtype(q, cos, sin)
    cos2, sin2, per_token = _rope_tables("attn_bwd_rope", cos, sin, head_dim, seq_len, batch * seq_len)
    _lib.call("fh_attn_bwd_rope", *args, _ptr(cos2), _ptr(sin2), per_token, _stream(q))


# ----------------------------------------------------- attention under a mask
def _int64_vector(name: str, t: torch.Tensor, n: int | None, dev: int) -> None:
    if t.get_device() != dev or dev < 0:
        raise ValueError(f"{name} must be on the mask's HIP device (femtohip ops take HIP device tensors only)")
    if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous int64 vector, got {t.dtype} {tuple(t.shape)}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} must have one entry a document, {n}, got {t.numel()}")


def attn_mask(tokens: int, seq_len: int, starts: torch.Tensor | None, lengths: torch.Tensor | None,
              prefix: torch.Tensor | None, window: int, causal: bool, device: torch.device) -> torch.Tensor:
    """The table of what each of `tokens` rows sees (fh_attn_mask): documents at rows starts
    (int64, ascending) of lengths (None: up to the next), or, starts None, one for each
    seq_len rows; window 0: none."""
    dev = device.index if device.index is not None else torch.cuda.current_device()
    n = starts.numel() if starts is not None else tokens // seq_len if seq_len else 0
    if starts is not None:
        _int64_vector("attention_mask: starts", starts, None, dev)
    for t, name in ((lengths, "lengths"), (prefix, "prefix")):
        if t is not None:  # (rows of no tokens are as many as they are)
            _int64_vector("attention_mask: " + name, t, n if starts is not None or seq_len else None, dev)
    nbytes = _lib.lib().fh_attn_mask_size(tokens)
    table = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _launch("fh_attn_mask", table, _ptr(starts), _ptr(lengths), _ptr(prefix), n, tokens, seq_len, window, int(causal),
            _ptr(table))
    return table


def token_rows(t: torch.Tensor, seq_len: int) -> int:
    """The row stride of [tokens, width] or [batch, seq_len, width] as token rows that the
    attention kernels read in place (its width for one row, which has none); 0 where they
    cannot."""
    if t.dim() == 2:
        ld, unit = t.stride()
        rows = t.size(0)
    else:
        outer, ld, unit = t.stride()
        rows = t.size(0)
        if rows > 1 and seq_len > 1 and outer != seq_len * ld:
            return 0
        if seq_len == 1:
            ld = outer
        rows *= seq_len
    width = t.size(-1)
    if rows <= 1:
        ld = width
    return ld if unit == 1 and ld >= width and ld % 8 == 0 and t.data_ptr() % 16 == 0 else 0


def masked_attn_check(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                      slopes: torch.Tensor | None, tokens: int, head_dim: int) -> tuple[int, int, int]:
    """(dtype code, n_heads, n_kv_heads) of token-major q, k and v of `tokens` rows, checked."""
    _alike(q, k, v)
    dev = q.get_device()
    if table.get_device() != dev:
        _require_gpu(q, table)
    q_shape, k_shape = q.shape, k.shape
    wq, wk = q_shape[-1], k_shape[-1]
    if head_dim <= 0 or wq % head_dim or wk % head_dim or k_shape != v.shape or q_shape[:-1] != k_shape[:-1] \
            or q.numel() != tokens * wq:
        raise ValueError(f"{name}: q must be [{tokens}, heads * {head_dim}], k and v [{tokens}, kv heads * {head_dim}], "
                         f"got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if table.dtype != torch.uint8 or table.numel() != _lib.lib().fh_attn_mask_size(tokens):
        raise ValueError(f"{name}: the mask is not one of {tokens} tokens")
    n_heads = wq // head_dim
    if slopes is not None:
        if slopes.get_device() != dev:
            _require_gpu(q, slopes)
        if slopes.dtype != torch.float32 or slopes.numel() != n_heads or not slopes.is_contiguous():
            raise ValueError(f"{name}: slopes must be contiguous fp32 with one entry a query head, {n_heads}")
    return _dtype_code(q), n_heads, wk // head_dim


def masked_attn_fwd_checked(args: tuple, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                            slopes: torch.Tensor | None, need_grad: bool):
    """masked_attn_fwd of tensors that are known to fit; args: (dtype code, ldq, ldk, ldv, tokens,
    n_heads, n_kv_heads, head_dim, scale, cap).  o has q's shape."""
    dt, ldq, ldk, ldv, T, nh, nkv, hd, scale, cap = args
    o = q.new_empty(q.shape)
    lse = low = None
    if need_grad:
        lse = q.new_empty((nh, T), dtype=torch.float32)
        if dt == _lib.FH_BF16:
            low = q.new_empty(q.shape, dtype=torch.int8)
    _launch("fh_masked_attn_fwd", q, dt, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, o.data_ptr(), nh * hd,
            _ptr(lse), _ptr(low), table.data_ptr(), T, nh, nkv, hd, scale, cap, _ptr(slopes))
    return o, lse, low


def masked_attn_bwd_checked(args: tuple, q, k, v, o, dout, lddo: int, lse, o_low, table, slopes):
    """masked_attn_bwd of tensors that are known to fit (o contiguous, dout of row stride lddo);
    args: masked_attn_fwd_checked's.  dq, dk, dv have q's, k's and v's shapes."""
    dt, ldq, ldk, ldv, T, nh, nkv, hd, scale, cap = args
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    ws = q.new_empty(max(_lib.lib().fh_masked_attn_bwd_workspace_size(dt, T, nh, nkv, hd), 4), dtype=torch.uint8)
    _launch("fh_masked_attn_bwd", q, dt, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, o.data_ptr(), nh * hd,
            dout.data_ptr(), lddo, lse.data_ptr(), _ptr(o_low), dq.data_ptr(), nh * hd, dk.data_ptr(), nkv * hd, dv.data_ptr(),
            nkv * hd, table.data_ptr(), ws.data_ptr(), T, nh, nkv, hd, scale, cap, _ptr(slopes))
    return dq, dk, dv


def _ld_of(name: str, **tensors: torch.Tensor) -> list[int]:
    lds = [token_rows(t, 0) if t.dim() == 2 else 0 for t in tensors.values()]
    for n, ld in zip(tensors, lds):
        if not ld:
            raise ValueError(f"{name}: {n} must be 2-D token rows, 16-byte aligned, its last dim contiguous and its row "
                             "stride a multiple of 8")
    return lds


def masked_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *, head_dim: int,
                    scale: float, cap: float = 0.0, slopes: torch.Tensor | None = None,
                    need_grad: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Attention of token-major q [T, heads * head_dim] over k and v [T, kv heads * head_dim]
    under attn_mask's table (fh_masked_attn_fwd): (o, lse, o_low), the latter two what
    masked_attn_bwd reads (None without need_grad; o_low of bf16 only).  cap 0: scores are
    not capped."""
    T = q.size(0)
    dt, nh, nkv = masked_attn_check("masked_attn_fwd", q, k, v, table, slopes, T, head_dim)
    lds = _ld_of("masked_attn_fwd", q=q, k=k, v=v)
    return masked_attn_fwd_checked((dt, *lds, T, nh, nkv, head_dim, scale, cap), q, k, v, table, slopes, need_grad)


def masked_attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, dout: torch.Tensor,
                    lse: torch.Tensor, o_low: torch.Tensor | None, table: torch.Tensor, *, head_dim: int, scale: float,
                    cap: float = 0.0, slopes: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of masked_attn_fwd for dout, with its o, lse and o_low: (dq, dk, dv)."""
    T = q.size(0)
    dt, nh, nkv = masked_attn_check("masked_attn_bwd", q, k, v, table, slopes, T, head_dim)
    ldq, ldk, ldv, lddo = _ld_of("masked_attn_bwd", q=q, k=k, v=v, dout=dout)
    _alike(q, o, dout)
    if o.shape != q.shape or dout.shape != q.shape or not o.is_contiguous():
        raise ValueError("masked_attn_bwd: o and dout must have q's shape, and o be contiguous")
    if lse.get_device() != q.get_device() or lse.dtype != torch.float32 or lse.numel() != nh * T or not lse.is_contiguous():
        raise ValueError("masked_attn_bwd: lse must be contiguous fp32 [heads, tokens]")
    if (o_low is None) == (dt == _lib.FH_BF16):
        raise ValueError("masked_attn_bwd: o_low goes with bf16")
    if o_low is not None and (o_low.get_device() != q.get_device() or o_low.dtype != torch.int8 or o_low.shape != q.shape
                              or not o_low.is_contiguous()):
        raise ValueError("masked_attn_bwd: o_low must be contiguous int8 of q's shape")
    return masked_attn_bwd_checked((dt, ldq, ldk, ldv, T, nh, nkv, head_dim, scale, cap), q, k, v, o, dout, lddo, lse, o_low,
                                   table, slopes)


def _cache_strides(name: str, t: torch.Tensor, batch: int, head_dim: int) -> tuple[int, int, int, int, int]:
    """(room, kv heads, batch stride, row stride, head stride) of a cache [batch, room, kv heads *
    head_dim] or [batch, room, kv heads, head_dim]; the stride of a dim of one is anything."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3 and shape[0] == batch and shape[2] % head_dim == 0:
        _, room, width = shape
        sb, sr, unit = stride
        heads, sh = width // head_dim, head_dim
    elif len(shape) == 4 and shape[0] == batch and shape[3] == head_dim:
        _, room, heads, _ = shape
        sb, sr, sh, unit = stride
    else:
        raise ValueError(f"cache_attn: {name} must be [{batch}, room, kv heads * {head_dim}] or [{batch}, room, kv heads, "
                         f"{head_dim}], got {tuple(shape)}")
    if unit != 1:
        raise ValueError(f"cache_attn: {name}'s last dim must be contiguous, got strides {stride}")
    return room, heads, sb if batch > 1 else 0, sr if room > 1 else head_dim, sh if heads > 1 else 0


def cache_attn(q: torch.Tensor, ldq: int, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, *, head_dim: int,
               scale: float, cap: float = 0.0, slopes: torch.Tensor | None = None, window: int = 0) -> torch.Tensor:
    """Attention of q [batch, n_new, heads * head_dim] (token rows of stride ldq) over caches k and v
    (_cache_strides), the new tokens being each sequence's last of lengths (int64 [batch])
    places (fh_cache_attn)."""
    _alike(q, k, v)
    dev = q.get_device()
    batch, n_new, width = q.shape
    room, nkv, kb, kr, kh = _cache_strides("k", k, batch, head_dim)
    room2, nkv2, vb, vr, vh = _cache_strides("v", v, batch, head_dim)
    if room2 != room or nkv2 != nkv:
        raise ValueError(f"cache_attn: k and v are {tuple(k.shape)} and {tuple(v.shape)}")
    if width % head_dim:
        raise ValueError(f"cache_attn: q must be [{batch}, new, heads * {head_dim}], got {tuple(q.shape)}")
    nh = width // head_dim
    if lengths.get_device() != dev:
        _require_gpu(q, lengths)
    if lengths.dtype != torch.int64 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError(f"cache_attn: lengths must be contiguous int64 [{batch}], got {lengths.dtype} {tuple(lengths.shape)}")
    if slopes is not None:
        if slopes.get_device() != dev:
            _require_gpu(q, slopes)
        if slopes.dtype != torch.float32 or slopes.numel() != nh or not slopes.is_contiguous():
            raise ValueError(f"cache_attn: slopes must be contiguous fp32 with one entry a query head, {nh}")
    dt = _dtype_code(q)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nbytes = _lib.lib().fh_cache_attn_workspace_size(dt, batch, n_new, room, nh, nkv, head_dim)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch("fh_cache_attn", q, dt, q.data_ptr(), ldq, k.data_ptr(), kb, kr, kh, v.data_ptr(), vb, vr, vh, o.data_ptr(), width,
            lengths.data_ptr(), batch, n_new, room, nh, nkv, head_dim, window, scale, cap, _ptr(slopes), _ptr(ws))
    return o


# ------------------------------------------------------------- loss head
def ce_fwd_bwd_(logits: torch.Tensor, labels: torch.Tensor, inv_count: torch.Tensor,
                ignore_index: int = -100) -> torch.Tensor:
    """Cross-entropy of the rows of `logits` [rows, V] against `labels` (int64
    [rows]); overwrites `logits` with the gradient (softmax - onehot) * inv_count
    (0 for ignored rows) and returns the fp32 per-row losses.  `inv_count` is a
    device fp32 scalar, 1 / (number of non-ignored labels of the whole batch)."""
    _require_gpu(logits, labels, inv_count)
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("ce_fwd_bwd_: logits must be a row-major 2-D tensor")
    if labels.dtype != torch.int64 or not labels.is_contiguous() or labels.numel() != logits.size(0):
        raise ValueError("ce_fwd_bwd_: labels must be contiguous int64 with one entry per row")
    if inv_count.dtype != torch.float32 or inv_count.numel() != 1:
        raise ValueError("ce_fwd_bwd_: inv_count must be a one-element fp32 tensor")
    loss_rows = torch.empty(logits.size(0), dtype=torch.float32, device=logits.device)
    _lib.call("fh_ce_fwd_bwd", _dtype_code(logits), _ptr(logits), logits.stride(0), _ptr(labels),
              logits.size(0), logits.size(1), int(ignore_index), _ptr(inv_count), _fptr(loss_rows),
              _stream(logits))
    return loss_rows


# ------------------------------------------------------------- embedding
def _embedding_args(weight: torch.Tensor, ids: torch.Tensor) -> tuple[int, int]:
    if weight.dim() != 2 or not weight.is_contiguous():
        raise ValueError("embedding: weight must be a contiguous [vocab, hidden] tensor")
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        raise ValueError("embedding: ids must be contiguous int64")
    vocab, hidden = weight.shape
    if hidden % 8 != 0:
        raise ValueError(f"embedding: hidden must be a multiple of 8, got {hidden}")
    return vocab, hidden


def embedding_fwd(ids: torch.Tensor, weight: torch.Tensor, factor: float = 1.0) -> torch.Tensor:
    """factor * weight[ids] (rounded once) with zero rows for ids outside [0, vocab):
    [*ids.shape, hidden]."""
    _alike(weight)
    if ids.get_device() != weight.get_device():
        _require_gpu(ids, weight)
    vocab, hidden = _embedding_args(weight, ids)
    out = torch.empty(*ids.shape, hidden, dtype=weight.dtype, device=weight.device)
    _launch("fh_embedding_scaled_fwd", weight, _dtype_code(weight), _ptr(weight), _ptr(ids), _ptr(out), ids.numel(), vocab,
            hidden, factor)
    return out


def embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, vocab: int, padding_idx: int | None = None,
                  factor: float = 1.0) -> torch.Tensor:
    """Weight gradient of the lookup: [vocab, hidden], row v = factor times the sum of the dy
    rows of the tokens with id v (fp32, token order), zero for unused ids; tokens with
    an id outside [0, vocab) or equal to padding_idx contribute nothing."""
    _require_gpu(dy, ids)
    hidden = dy.size(-1)
    if not dy.is_contiguous() or dy.numel() != ids.numel() * hidden:
        raise ValueError("embedding_bwd: dy must be contiguous [*ids.shape, hidden]")
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        raise ValueError("embedding_bwd: ids must be contiguous int64")
    if hidden % 8 != 0:
        raise ValueError(f"embedding_bwd: hidden must be a multiple of 8, got {hidden}")
    dw = torch.empty(vocab, hidden, dtype=dy.dtype, device=dy.device)
    n = ids.numel()
    ws = torch.empty(_lib.lib().fh_embedding_bwd_workspace_size(n, vocab), dtype=torch.uint8,
                     device=dy.device)
    _launch("fh_embedding_scaled_bwd", dy, _dtype_code(dy), _ptr(dy), _ptr(ids), _ptr(dw), n, vocab, hidden,
            -1 if padding_idx is None else int(padding_idx), factor, _ptr(ws))
    return dw


# ------------------------------------------------------------- gradient norm
def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors of one shape lie alike; the stride of a dim of one is anything."""
    return all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


def clip_grads(grads: list, outs: list | None, max_norm: float) -> torch.Tensor:
    """The 2-norm of all grads (a one-element fp32 tensor) and, with outs, each of them times
    min(1, max_norm / (norm + 1e-6)) (fh_clip_grads).  Tensors are dense, an out of its
    gradient's strides, and on one device; an out may be its gradient."""
    first = grads[0]
    dev = first.get_device()
    in_place = outs is grads
    all_contiguous = True
    for ts in (grads,) if outs is None or in_place else (grads, outs):
        if dev < 0 or any([t.get_device() != dev for t in ts]):
            _require_gpu(first, *ts)
        if not all([t.layout == torch.strided and t.is_contiguous() for t in ts]):
            all_contiguous = False
            if not all([t.layout == torch.strided and torch.ops.aten.is_non_overlapping_and_dense(t) for t in ts]):
                raise ValueError("clip_gradients: gradients must be dense")
    if outs is not None and not in_place:
        if [t.shape for t in grads] != [t.shape for t in outs] \
                or not (all_contiguous or all([a.stride() == b.stride() or (a.is_contiguous() and b.is_contiguous())
                                               or _same_order(a, b) for a, b in zip(grads, outs)])):
            raise ValueError("clip_gradients: an output must have its gradient's shape and strides")
    n = len(grads)
    table = (_lib.FhGrad * n)()
    # an fh_grad as four 64-bit words: grad, out, numel, the dtypes
    words = (ctypes.c_uint64 * (4 * n)).from_buffer(table)
    words[0::4] = [t.data_ptr() for t in grads]
    if outs is not None:
        words[1::4] = words[0::4] if in_place else [t.data_ptr() for t in outs]
    words[2::4] = [t.numel() for t in grads]
    kinds = [_dtype_code(t) for t in grads]
    words[3::4] = [a | b << 32 for a, b in zip(kinds, kinds if outs is None or in_place else map(_dtype_code, outs))]
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    ws = torch.empty(_lib.lib().fh_clip_grads_workspace_size(n), dtype=torch.uint8, device=first.device)
    _launch("fh_clip_grads", first, n, ctypes.addressof(table), max_norm, norm.data_ptr(), ws.data_ptr())
    return norm


# ------------------------------------------------------------- decoder layer
def layer_args(batch: int, seq_len: int, shp, dtype: torch.dtype) -> _lib.FhLayer | None:
    """The sizes of an fh_layer argument block, of a layer of shape `shp`
    (fused_layer.LayerShape), which layer_workspace_size reads; None for a dtype
    that the layer calls do not take.  layer_operands adds the pointers."""
    if dtype not in _DT:
        return None
    return _lib.FhLayer(_DT[dtype], 0, batch, seq_len, shp.hidden, shp.n_heads, shp.n_kv_heads, shp.head_dim, shp.ffn,
                        shp.eps1, shp.eps2, shp.scale)


def layer_operands(args: _lib.FhLayer, shp, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *ws: torch.Tensor):
    """Points the block of layer_args at the operands of x's layer, with weights
    wqkv, wo, wgu, wd, w1, w2, and returns the tensors that it then points into;
    None where an operand is not what the layer calls take: x's device and dtype,
    contiguous, 16-byte aligned, of the shape's sizes.  The caller keeps the
    tensors alive and uses the block at once."""
    H, hq, F_ = shp.hidden, shp.hq, shp.ffn
    sizes = ((hq + 2 * shp.hkv, H), (H, hq), (2 * F_, H), (H, F_), (H,), (H,))
    dt, dev = x.dtype, x.device
    for w, size in zip(ws, sizes):
        if w.dtype != dt or w.device != dev or w.shape != size or not w.is_contiguous() or w.data_ptr() % 16:
            return None
    if not x.is_cuda or not x.is_contiguous() or x.data_ptr() % 16:
        return None
    if not cos.dtype == sin.dtype == dt or not cos.device == sin.device == dev:
        return None
    cos2, sin2, per_token = _rope_tables("layer", cos, sin, shp.head_dim, args.seq_len, args.batch * args.seq_len)
    args.cos_per_token, args.cos, args.sin = per_token, cos2.data_ptr(), sin2.data_ptr()
    args.wqkv, args.wo, args.wgu, args.wd, args.w1, args.w2 = (w.data_ptr() for w in ws)
    return (cos2, sin2, *ws)


def layer_workspace_size(args: _lib.FhLayer, backward: bool) -> int:
    return _lib.lib().fh_layer_workspace_size(ctypes.byref(args), int(backward))


def layer_fwd(args: _lib.FhLayer, nbytes: int, x: torch.Tensor) -> torch.Tensor:
    """fh_layer_fwd on the x of layer_operands, with a workspace of nbytes."""
    out = torch.empty_like(x)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.call("fh_layer_fwd", ctypes.byref(args), x.data_ptr(), out.data_ptr(), ws.data_ptr(), _stream(x))
    return out


def layer_bwd(args: _lib.FhLayer, nbytes: int, x: torch.Tensor, dout: torch.Tensor, grads: list,
              accumulate: int) -> torch.Tensor:
    """fh_layer_bwd on contiguous, 16-byte aligned x and dout; grads: the dwqkv, dwo, dwgu, dwd, dw1, dw2 buffers.  Returns dx."""
    dx = torch.empty_like(x)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.call("fh_layer_bwd", ctypes.byref(args), x.data_ptr(), dout.data_ptr(), dx.data_ptr(),
              *(g.data_ptr() for g in grads), accumulate, ws.data_ptr(), _stream(x))
    return dx


# ------------------------------------------------------------- GEMM
_GEMM_OPS = {"nt": _lib.FH_GEMM_NT, "nn": _lib.FH_GEMM_NN, "tn": _lib.FH_GEMM_TN}


def gemm_dims(op: str, a: torch.Tensor, b: torch.Tensor):
    """(m, n, k) of op(a) @ op(b), or None if the shapes do not chain."""
    if a.dim() != 2 or b.dim() != 2:
        return None
    if op == "nt":
        (m, k), (n, kb) = a.shape, b.shape
    elif op == "nn":
        (m, k), (kb, n) = a.shape, b.shape
    elif op == "tn":
        (k, m), (kb, n) = a.shape, b.shape
    else:
        raise ValueError(f"gemm: op must be 'nt', 'nn' or 'tn', got {op!r}")
    return (m, n, k) if k == kb else None


def gemm_supported(op: str, a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether fh_gemm_bf16 takes these operands: bf16 on one HIP device, 2-D
    with a contiguous last dim, k a multiple of 64, n (and for 'tn' also m) a
    multiple of 8, row strides multiples of 8 and 16-byte aligned data."""
    return _gemm_operands_ok(op, a, b, False)


def gemm_any_k_supported(op: str, a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether fh_gemm_bf16_any_k takes these operands: as gemm_supported, but
    any k of at least 64 ('tn'), or its multiples of 8 ('nt', 'nn')."""
    return _gemm_operands_ok(op, a, b, True)


def _gemm_operands_ok(op: str, a: torch.Tensor, b: torch.Tensor, any_k: bool) -> bool:
    if not (a.is_cuda and b.is_cuda and a.device == b.device and a.dtype == b.dtype == torch.bfloat16):
        return False
    dims = gemm_dims(op, a, b)
    if dims is None:
        return False
    m, n, k = dims
    if min(m, n, k) <= 0 or n % 8 or (op == "tn" and m % 8):
        return False
    if k % 64 and not (any_k and k >= 64 and (op == "tn" or k % 8 == 0)):
        return False
    for t in (a, b):
        if t.stride(1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16:
            return False
    return True


def gemm(op: str, a: torch.Tensor, b: torch.Tensor, *, residual: torch.Tensor | None = None,
         out: torch.Tensor | None = None, any_k: bool = False) -> torch.Tensor:
    """op(a) @ op(b) in bf16 with fp32 accumulation (fh_gemm_bf16):
    'nt': a [m,k] @ b[n,k]^T (nn.Linear forward), 'nn': a [m,k] @ b [k,n]
    (input gradient), 'tn': a[k,m]^T @ b [k,n] (weight gradient).  With
    `residual` ([m, n]) returns residual + to_bf16(product), rounded again;
    `out` may be `residual` itself.  `any_k`: k need not be a multiple of 64
    (fh_gemm_bf16_any_k, gemm_any_k_supported)."""
    _require_gpu(a, b, residual, out)
    if not _gemm_operands_ok(op, a, b, any_k):
        raise ValueError(f"gemm({op}): unsupported operands {tuple(a.shape)} {a.stride()} x "
                         f"{tuple(b.shape)} {b.stride()} ({a.dtype}, {b.dtype})")
    m, n, k = gemm_dims(op, a, b)
    c = torch.empty(m, n, dtype=a.dtype, device=a.device) if out is None else out
    for t, name in ((c, "out"), (residual, "residual")):
        if t is None:
            continue
        if t.dtype != torch.bfloat16 or tuple(t.shape) != (m, n) or t.stride(1) != 1:
            raise ValueError(f"gemm({op}): {name} must be a bf16 [{m}, {n}] row-major view")
        if t.stride(0) % 8 or t.data_ptr() % 16:
            raise ValueError(f"gemm({op}): {name} must be 16-byte aligned with a row stride % 8 == 0")
    code = _GEMM_OPS[op]
    name = "fh_gemm_bf16_any_k" if any_k else "fh_gemm_bf16"
    nbytes = getattr(_lib.lib(), name + "_workspace_size")(code, m, n, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device) if nbytes else None
    _lib.call(name, code, _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(c), c.stride(0),
              _ptr(residual), 0 if residual is None else residual.stride(0), m, n, k, _ptr(ws),
              _stream(a))
    return c


def gemm_acc(a: torch.Tensor, b: torch.Tensor, acc: torch.Tensor, *, add: bool,
             out: torch.Tensor | None = None) -> None:
    """acc (fp32 [m, n], contiguous) = a[k,m]^T @ b[k,n] (+ acc, with `add`), in
    fp32; with `out` (bf16 [m, n]) the sum is rounded into `out` instead and acc
    only read (fh_gemm_bf16_acc)."""
    _require_gpu(a, b, acc, out)
    if not gemm_any_k_supported("tn", a, b):
        raise ValueError(f"gemm_acc: unsupported operands {tuple(a.shape)} {a.stride()} x {tuple(b.shape)} {b.stride()}")
    m, n, k = gemm_dims("tn", a, b)
    if acc.dtype != torch.float32 or acc.shape != (m, n) or not acc.is_contiguous() or acc.data_ptr() % 16:
        raise ValueError(f"gemm_acc: acc must be an aligned, contiguous fp32 [{m}, {n}] tensor")
    if out is not None and (out.dtype != torch.bfloat16 or out.shape != (m, n) or out.stride(1) != 1
                            or out.stride(0) % 8 or out.data_ptr() % 16):
        raise ValueError(f"gemm_acc: out must be a 16-byte aligned bf16 [{m}, {n}] view, row stride % 8 == 0")
    _lib.call("fh_gemm_bf16_acc", _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(acc), int(add), _ptr(out),
              0 if out is None else out.stride(0), m, n, k, _stream(a))


# fh_gemm_f32 takes products of at most this many outputs and k (weight
# gradients: k of at most 256).  There the library runs some shapes as one tile
# on one CU (256 x 256 x 688 160 us against 8, 256 x 256 x 512 'nn' 118 against 8)
# and the others within 1 us of it (5-8 us); above, its choices are sound and its
# tiles faster (512 x 1376 x 256 7.5 us against 9.9, 2048 x 256 x 688 12 against 14).
F32_MAX_OUTPUTS = 98304
F32_MAX_K = {"nt": 768, "nn": 768, "tn": 256}


def gemm_f32_supported(op: str, a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a product runs on fh_gemm_f32: fp32 on one HIP device, 2-D with a
    contiguous last dim, small (above), and where k is an operand's last dim,
    multiples of 4 and 16-byte aligned rows."""
    if not (a.is_cuda and b.is_cuda and a.device == b.device and a.dtype == b.dtype == torch.float32):
        return False
    dims = gemm_dims(op, a, b)
    if dims is None:
        return False
    m, n, k = dims
    if min(m, n, k) <= 0 or m * n > F32_MAX_OUTPUTS or k > F32_MAX_K[op]:
        return False
    for t, k_last in ((a, op != "tn"), (b, op == "nt")):
        if t.stride(1) != 1 or t.stride(0) < t.size(1) or (k_last and (k % 4 or t.stride(0) % 4 or t.data_ptr() % 16)):
            return False
    return True


def gemm_f32(op: str, a: torch.Tensor, b: torch.Tensor, *, residual: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """gemm() in fp32 for small products (fh_gemm_f32): op(a) @ op(b), plus
    `residual`, into `out` (which may be `residual` itself)."""
    _require_gpu(a, b, residual, out)
    if not gemm_f32_supported(op, a, b):
        raise ValueError(f"gemm_f32({op}): unsupported operands {tuple(a.shape)} {a.stride()} x "
                         f"{tuple(b.shape)} {b.stride()} ({a.dtype}, {b.dtype})")
    m, n, k = gemm_dims(op, a, b)
    c = torch.empty(m, n, dtype=a.dtype, device=a.device) if out is None else out
    for t, name in ((c, "out"), (residual, "residual")):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (m, n) or t.stride(1) != 1):
            raise ValueError(f"gemm_f32({op}): {name} must be an fp32 [{m}, {n}] row-major view")
    _lib.call("fh_gemm_f32", _GEMM_OPS[op], _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(c), c.stride(0),
              _ptr(residual), 0 if residual is None else residual.stride(0), m, n, k, _stream(a))
    return c


def gemm_grouped(op: str, items: list, *, any_k: bool = False) -> list:
    """Up to three GEMMs of layout `op` with one k in one fh_gemm_bf16_grouped
    call: each item is (a, b, residual, out) with gemm()'s meaning (residual
    and out may be None; out may be residual itself), `any_k` too.  Returns the
    outputs."""
    if not 1 <= len(items) <= 3:
        raise ValueError(f"gemm_grouped({op}): between 1 and 3 problems, got {len(items)}")
    probs = (_lib.FhGemmProblem * len(items))()
    outs, ks = [], set()
    for i, (a, b, residual, out) in enumerate(items):
        _require_gpu(a, b, residual, out)
        if not _gemm_operands_ok(op, a, b, any_k):
            raise ValueError(f"gemm_grouped({op}): unsupported operands {tuple(a.shape)} {a.stride()} x "
                             f"{tuple(b.shape)} {b.stride()} ({a.dtype}, {b.dtype})")
        m, n, k = gemm_dims(op, a, b)
        ks.add(k)
        c = torch.empty(m, n, dtype=a.dtype, device=a.device) if out is None else out
        for t, name in ((c, "out"), (residual, "residual")):
            if t is None:
                continue
            if t.dtype != torch.bfloat16 or tuple(t.shape) != (m, n) or t.stride(1) != 1:
                raise ValueError(f"gemm_grouped({op}): {name} must be a bf16 [{m}, {n}] row-major view")
            if t.stride(0) % 8 or t.data_ptr() % 16:
                raise ValueError(f"gemm_grouped({op}): {name} must be 16-byte aligned with a row stride % 8 == 0")
        probs[i] = _lib.FhGemmProblem(_ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(c), c.stride(0),
                                      _ptr(residual), 0 if residual is None else residual.stride(0), m, n)
        outs.append(c)
    if len(ks) != 1:
        raise ValueError(f"gemm_grouped({op}): the problems' k differ: {sorted(ks)}")
    k = ks.pop()
    code = _GEMM_OPS[op]
    a0 = items[0][0]
    if any(t is not None and t.device != a0.device for item in items for t in item) or \
            any(o.device != a0.device for o in outs):
        raise ValueError(f"gemm_grouped({op}): every operand and output must be on {a0.device}")
    name = "fh_gemm_bf16_grouped_any_k" if any_k else "fh_gemm_bf16_grouped"
    nbytes = getattr(_lib.lib(), name + "_workspace_size")(code, len(items), probs, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=a0.device) if nbytes else None
    _lib.call(name, code, len(items), probs, k, _ptr(ws), _stream(a0))
    return outs


def gemm_rope(a: torch.Tensor, b: torch.Tensor, n_rot_heads: int, head_dim: int, seq_len: int,
              cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """a [m,k] @ b[n,k]^T (the q/k/v projection) with the rotary embedding of
    rope_fwd_ applied to heads 0..n_rot_heads-1 of the output in the GEMM's
    epilogue (fh_gemm_bf16_rope); rows of a are tokens."""
    _require_gpu(a, b, cos, sin)
    if not gemm_supported("nt", a, b):
        raise ValueError(f"gemm_rope: unsupported operands {tuple(a.shape)} {a.stride()} x "
                         f"{tuple(b.shape)} {b.stride()} ({a.dtype}, {b.dtype})")
    _same_dtype(a, cos, sin)
    m, n, k = gemm_dims("nt", a, b)
    cos2, sin2, per_token = _rope_tables("gemm_rope", cos, sin, head_dim, seq_len, m)
    c = torch.empty(m, n, dtype=a.dtype, device=a.device)
    _lib.call("fh_gemm_bf16_rope", _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(c), c.stride(0),
              m, n, k, n_rot_heads * head_dim, head_dim, seq_len, _ptr(cos2), _ptr(sin2), per_token,
              _stream(a))
    return c


