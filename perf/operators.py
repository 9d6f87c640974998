"""The operators around a checkpointed block whose speed is followed: their cases,
their plain forms and their values in 64 bits.

* ``store``: an activation kept in 8 bits and read back (what a checkpointed
  MLP does with its input), ``norm8``: a checkpointed RMSNorm that keeps its
  input in 8 bits, forward and backward; ``recompute8``: the two norms of a
  checkpointed layer's recompute, read from the kept input.
* ``norms``: the norms after and before a block with the block's gate and
  residual scale, forward alone or with its backward.
* ``rotary``: rotary positions of q and k, forward alone or with the backward.

Widths are those of the repository's configurations (hidden 256, 2048, 4096; 32
query heads over 4, 8 or 32 kv heads of 64 or 128) and odd ones (688, the debug
model's ffn; 1000), token counts run from one to the longest configured one.

8-bit storage: blocks of 32 elements of a row (the row's last one may be
shorter) share an exponent E, kept as the byte E + 127, and an element is
code * 2^E.  With e the exponent of the block's largest magnitude m (2^e <= m <
2^(e+1)): int8 has E = e - 6 and code = round(x 2^-E), at most 127 in
magnitude; e4m3 has E = e - 8, one more where m 2^-E would pass 448, and code =
x 2^-E rounded to e4m3.  E is at least -118.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 32
MIN_E = -118


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One short sequence of a checkpointed norm: launches are the time.
        dict(name="norm8_short", kind="norm8", fmt="int8", tokens=256, hidden=2048, dtype="bf16", dres=False),
        # The configured TinyLlama step's norm with the residual gradient beside it.
        dict(name="norm8_train", kind="norm8", fmt="int8", tokens=16384, hidden=2048, dtype="bf16", dres=True),
        # An odd width and token count in fp32: the debug model's ragged batch.
        dict(name="norm8_ragged_fp32", kind="norm8", fmt="e4m3", tokens=999, hidden=688, dtype="fp32", dres=True),
        # The recompute of an 8B-wide layer at its configured 8192 tokens.
        dict(name="recompute8_8b", kind="recompute8", fmt="e4m3", tokens=8192, hidden=4096, dtype="bf16"),
        # A checkpointed MLP's input at the long-context configuration.
        dict(name="store_long", kind="store", fmt="int8", tokens=32768, hidden=4096, dtype="bf16"),
        # A single token while answering: the norms between two blocks.
        dict(name="norms_token", kind="norms", way="fwd", gate="channel", post=True, pre=True, scale=1.0,
             tokens=1, hidden=4096, dtype="bf16"),
        # The training step's width with a learned gate per channel.
        dict(name="norms_train", kind="norms", way="both", gate="channel", post=True, pre=True, scale=0.5,
             tokens=16384, hidden=2048, dtype="bf16"),
        # A ragged batch with a gate that each token computes.
        dict(name="norms_ragged", kind="norms", way="both", gate="token", post=True, pre=True, scale=1.0,
             tokens=999, hidden=2048, dtype="bf16"),
        # The 8B width with a residual multiplier and no norm after the block.
        dict(name="norms_8b", kind="norms", way="both", gate="none", post=False, pre=True, scale=0.22,
             tokens=8192, hidden=4096, dtype="bf16"),
        # A few tokens while answering, far into a stretched context.
        dict(name="rotary_token", kind="rotary", way="fwd", layout="half", tokens=4, heads=32, kv=8, head_dim=128,
             rot=128, offset=0, theta=5e5, scaling="llama3", first=100000, dtype="bf16"),
        # The training step's heads, positions starting anew with each packed sequence.
        dict(name="rotary_train", kind="rotary", way="both", layout="half", tokens=16384, heads=32, kv=4, head_dim=64,
             rot=64, offset=0, theta=1e4, scaling="none", first=0, dtype="bf16"),
        # Half of each head, neighbouring pairs, at the long-context configuration.
        dict(name="rotary_long", kind="rotary", way="both", layout="interleaved", tokens=32768, heads=32, kv=32,
             head_dim=128, rot=64, offset=64, theta=1e4, scaling="yarn", first=0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm8", "recompute8", "store", "norms", "norms", "rotary", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    tokens = _log(rng, 1, 32768)
    most = (1 << 26) // (2 if dtype == "fp32" else 1)
    if kind == "rotary":
        head_dim = rng.choice([32, 64, 80, 96, 128, 256])
        rot = rng.choice([head_dim, head_dim // 2, 16])
        heads = rng.choice([1, 5, 8, 32])
        kv = rng.choice([1, 4, 8, heads])
        return dict(kind=kind, way=rng.choice(["fwd", "both"]), layout=rng.choice(["half", "interleaved"]),
                    tokens=max(1, min(tokens, most // ((heads + kv) * head_dim))), heads=heads, kv=kv,
                    head_dim=head_dim, rot=rot, offset=rng.choice([0, head_dim - rot]),
                    theta=rng.choice([1e4, 5e5]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                    first=rng.choice([0, _log(rng, 1, 1 << 20)]), dtype=dtype)
    hidden = rng.choice([256, 688, 1000, 2048, 4096, 8 * _log(rng, 1, 1024)])
    tokens = max(1, min(tokens, most // hidden))
    if kind == "norms":
        post, pre = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return dict(kind=kind, way=rng.choice(["fwd", "both", "both"]), gate=rng.choice(["none", "channel", "token"]),
                    post=post, pre=pre, scale=rng.choice([1.0, 0.5, 0.22]), tokens=tokens, hidden=hidden, dtype=dtype)
    case = dict(kind=kind, fmt=rng.choice(["int8", "e4m3"]), tokens=tokens, hidden=hidden, dtype=dtype)
    if kind == "norm8":
        case["dres"] = rng.choice([True, False])
    return case


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=gen, device=DEV).mul_(std).add_(mean).to(dtype)


def _stream(gen, tokens, hidden, dtype):
    """A residual stream: a spread of row sizes and a few channels far above the rest."""
    x = torch.randn(tokens, hidden, generator=gen, device=DEV)
    x.mul_(torch.rand(tokens, 1, generator=gen, device=DEV).mul_(2).add_(0.5))
    big = torch.rand(hidden, generator=gen, device=DEV) < 0.005
    return x.mul_(torch.where(big, 40.0, 1.0)).to(dtype)


def _inv_freq(case):
    """Angle per position of each rotated pair, and the factor on cos and sin, in 64 bits."""
    n, theta, kind = case["rot"] // 2, case["theta"], case["scaling"]
    f = theta ** (-torch.arange(n, dtype=torch.float64) / n)
    turn = 2 * math.pi
    if kind == "linear":
        return f / 4.0, 1.0
    if kind == "llama3":  # long waves slowed 8 times, short ones kept, a ramp between
        wave = turn / f
        ramp = ((8192 / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * (ramp + (1 - ramp) / 8.0), 1.0
    if kind == "yarn":  # the ramp runs over pair indices, from 32 turns to 1 in 4096 positions
        at = [n * math.log(4096 / (b * turn)) / math.log(theta) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 2 * n - 1)
        ramp = 1 - ((torch.arange(n, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (ramp + (1 - ramp) / 8.0), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, T = DTYPES[case["dtype"]], case["tokens"]
    s = dict(case=case)
    if case["kind"] == "rotary":
        wq, wk = case["heads"] * case["head_dim"], case["kv"] * case["head_dim"]
        qkv = _normal(gen, T, wq + 2 * wk, dtype=dt)  # q and k are columns of the packed projection
        s["q"], s["k"] = qkv[:, :wq], qkv[:, wq:wq + wk]
        length = int(torch.randint(max(1, T // 8), T + 1, (1,), generator=gen, device=DEV))
        s["pos"] = torch.arange(T, device=DEV) % length + case["first"]
        s["inv_freq"], s["factor"] = _inv_freq(case)
        s["inv_freq"] = s["inv_freq"].to(DEV)
        s["dq"] = _normal(gen, T, wq, dtype=dt, std=0.01)
        s["dk"] = _normal(gen, T, wk, dtype=dt, std=0.01)
        return s
    H = case["hidden"]
    s["x"] = _stream(gen, T, H, dt)
    if case["kind"] == "norms":
        s["a"] = _normal(gen, T, H, dtype=dt, std=0.7)
        s["w_post"] = _normal(gen, H, dtype=dt, std=0.1, mean=1.0) if case["post"] else None
        s["w_pre"] = _normal(gen, H, dtype=dt, std=0.02, mean=1.0) if case["pre"] else None
        s["gate"] = None
        if case["gate"] == "channel":
            s["gate"] = _normal(gen, H, dtype=dt, std=0.1, mean=0.3)
        elif case["gate"] == "token":
            s["gate"] = torch.sigmoid(torch.randn(T, H, generator=gen, device=DEV)).to(dt)
        s["dh"] = _normal(gen, T, H, dtype=dt, std=0.01)
        s["dy"] = _normal(gen, T, H, dtype=dt, std=0.01) if case["pre"] else None
        for k in ("x", "a", "w_post", "w_pre", "gate"):
            if s[k] is not None and case["way"] == "both":
                s[k].requires_grad_(True)
        return s
    s["w"] = _normal(gen, H, dtype=dt, std=0.02, mean=1.0)
    if case["kind"] == "norm8":
        s["dy"] = _normal(gen, T, H, dtype=dt, std=0.01)
        s["dres"] = _normal(gen, T, H, dtype=dt, std=0.01) if case["dres"] else None
    elif case["kind"] == "recompute8":
        s["codes"], s["exps"] = _pack(s.pop("x"), case["fmt"])
        s["a"] = _normal(gen, T, H, dtype=dt, std=0.7)
        s["w2"] = _normal(gen, H, dtype=dt, std=0.02, mean=1.0)
    return s


# ------------------------------------------------------------------ plain forms
def _two(e):
    """2^e in fp32, of whole numbers e."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK)


def _pack(x, fmt):
    """codes [T, H] and exponent bytes [T, ceil(H / 32)] of x."""
    xb = _blocks(x.float())
    m = xb.abs().amax(-1)
    e = (m.view(torch.int32) >> 23) - 127
    if fmt == "int8":
        E = (e - 6).clamp_min(MIN_E)
        c = (xb * _two(-E)[..., None]).round_().clamp_(-127, 127).to(torch.int8)
    else:
        E = (e - 8).clamp_min(MIN_E)
        E = E + (m * _two(-E) > 448).int()
        c = (xb * _two(-E)[..., None]).to(torch.float8_e4m3fn)
    codes = c.view(x.shape[0], -1)[:, :x.shape[1]].contiguous()
    return codes, (E + 127).to(torch.uint8)


def _unpack(codes, exps):
    E = exps.to(torch.int32).sub_(127).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float().mul_(_two(E))


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _norm_grad(dy, x, w):
    """The gradient of _norm with respect to x, and x over its root mean square."""
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n, g = x * r, dy * w
    return r * (g - n * (g * n).mean(-1, keepdim=True)), n


def _plain_norms(s):
    c, dt = s["case"], s["x"].dtype
    f = {k: v.detach().float() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    one = torch.ones((), device=DEV)
    x, a, scale = f["x"], f["a"], c["scale"]
    gate = one if f["gate"] is None else f["gate"]
    n = _norm(a, f["w_post"]) if c["post"] else a
    h = (x + scale * gate * n).to(dt)
    out = {"h": h}
    if c["pre"]:
        out["y"] = _norm(h.float(), f["w_pre"]).to(dt)
    if c["way"] == "fwd":
        return out
    D = f["dh"]
    if c["pre"]:
        g, nh = _norm_grad(f["dy"], h.float(), f["w_pre"])
        D = D + g
        out["dw_pre"] = (f["dy"] * nh).sum(0).to(dt)
    out["dx"] = D.to(dt)
    P = scale * gate * D
    if c["post"]:
        da, na = _norm_grad(P, a, f["w_post"])
        out["da"], out["dw_post"] = da.to(dt), (P * na).sum(0).to(dt)
    else:
        out["da"] = P.to(dt)
    if c["gate"] != "none":
        dg = scale * D * n
        out["dgate"] = (dg.sum(0) if c["gate"] == "channel" else dg).to(dt)
    return out


def _turn(x, cos, sin, case):
    """The rotated dims of each head turned; cos and sin are [T, 1, rot / 2]."""
    T, n = x.shape[0], case["rot"] // 2
    out = x.float().reshape(T, -1, case["head_dim"]).clone()
    part = out[..., case["offset"]:case["offset"] + case["rot"]]
    if case["layout"] == "half":
        u, v = part[..., :n], part[..., n:]
    else:
        u, v = part[..., 0::2], part[..., 1::2]
    nu, nv = u * cos - v * sin, v * cos + u * sin
    u.copy_(nu)
    v.copy_(nv)
    return out.view(T, -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    angle = s["pos"].double()[:, None, None] * s["inv_freq"]
    cos = (angle.cos() * s["factor"]).float()
    sin = (angle.sin() * s["factor"]).float()
    out = {"q": _turn(s["q"], cos, sin, c), "k": _turn(s["k"], cos, sin, c)}
    if c["way"] == "both":
        out["dq"], out["dk"] = _turn(s["dq"], cos, -sin, c), _turn(s["dk"], cos, -sin, c)
    return out


def _plain(s):
    c = s["case"]
    kind, dt = c["kind"], DTYPES[c["dtype"]]
    if kind == "norms":
        return _plain_norms(s)
    if kind == "rotary":
        return _plain_rotary(s)
    if kind == "store":
        return {"x": _unpack(*_pack(s["x"], c["fmt"])).to(dt)}
    w = s["w"].float()
    if kind == "recompute8":
        x = _unpack(s["codes"], s["exps"])
        h = (x + s["a"].float()).to(dt)
        return {"y": _norm(x, w).to(dt), "h": h, "z": _norm(h.float(), s["w2"].float()).to(dt)}
    y = _norm(s["x"].float(), w).to(dt)
    x = _unpack(*_pack(s["x"], c["fmt"]))
    dy = s["dy"].float()
    dx, n = _norm_grad(dy, x, w)
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"y": y, "dx": dx.to(dt), "dw": (dy * n).sum(0).to(dt)}


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from femtotron_amd import apply_rotary, block_norms, ops
    c = s["case"]
    kind = c["kind"]
    if kind == "norms":
        args = (s["x"], s["a"], s["w_post"], s["w_pre"])
        h, y = block_norms(*args, gate=s["gate"], scale=c["scale"], eps=EPS)
        out = {"h": h.detach()}
        if y is not None:
            out["y"] = y.detach()
        if c["way"] == "both":
            names = [k for k in ("x", "a", "w_post", "w_pre", "gate") if s[k] is not None]
            outs, grads = ((h,), (s["dh"],)) if y is None else ((h, y), (s["dh"], s["dy"]))
            for k, g in zip(names, torch.autograd.grad(outs, [s[k] for k in names], grads)):
                out["d" + k] = g
        return out
    if kind == "rotary":
        how = dict(head_dim=c["head_dim"], rot_dim=c["rot"], offset=c["offset"], layout=c["layout"], factor=s["factor"])
        if c["way"] == "fwd":
            q, k = apply_rotary(s["q"], s["k"], s["pos"], s["inv_freq"], **how)
            return {"q": q, "k": k}
        q, k = ops.rotary_fwd(s["q"], s["k"], s["pos"], s["inv_freq"], **how)
        dq, dk = ops.rotary_bwd(s["dq"], s["dk"], s["pos"], s["inv_freq"], **how)
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if kind == "store":
        return {"x": ops.unpack8(ops.pack8(s["x"], c["fmt"]), s["x"].dtype)}
    if kind == "recompute8":
        kept = ops.Packed8(s["codes"], s["exps"])
        y = ops.rmsnorm_fwd8(kept, s["w"], EPS)
        h, z = ops.add_rmsnorm_fwd8(kept, s["a"], s["w2"], EPS)
        return {"y": y, "h": h, "z": z}
    y, kept = ops.rmsnorm_fwd_pack8(s["x"], s["w"], EPS, c["fmt"])
    dx, dw = ops.rmsnorm_bwd8(s["dy"], kept, s["w"], EPS, dres=s["dres"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work
def work(case):
    """Each call of a pass reads its inputs and writes its outputs once: a backward
    is a call of its own, later, and reads again what the forward had."""
    size = DTYPES[case["dtype"]].itemsize
    T, kind = case["tokens"], case["kind"]
    if kind == "rotary":
        n = T * (case["heads"] + case["kv"]) * case["head_dim"]
        passes = 2 if case["way"] == "both" else 1
        turned = n * case["rot"] // case["head_dim"]
        return {"bytes": passes * (2 * n * size + 8 * T), "flops": passes * 3 * turned}
    H = case["hidden"]
    n = T * H
    kept = n + T * -(-H // BLOCK)
    if kind == "store":
        return {"bytes": 2 * n * size + 2 * kept, "flops": 4 * n}
    if kind == "norm8":
        passes = 5 if case["dres"] else 4  # x, y; dy, dx, dres
        return {"bytes": passes * n * size + 2 * kept + 3 * H * size, "flops": 18 * n}
    if kind == "recompute8":
        return {"bytes": 4 * n * size + kept + 2 * H * size, "flops": 11 * n}
    token = case["gate"] == "token"
    rows = 3 + case["pre"] + token
    vectors = case["post"] + case["pre"] + (case["gate"] == "channel")
    flops = n * (2 + 4 * case["post"] + 4 * case["pre"])
    if case["way"] == "both":
        # dh, dy, a (h too, for the norm before) in, dx and da out; the gate and its gradient
        rows += 4 + 2 * case["pre"] + 2 * token
        if not case["post"] and case["gate"] == "none":
            rows -= 1  # a's values are not needed
        flops += n * (4 + 8 * case["post"] + 10 * case["pre"])
        vectors *= 3
    return {"bytes": rows * n * size + vectors * H * size, "flops": flops}


# ------------------------------------------------------------------ values in 64 bits
def _power(e):
    """2^e in fp64, of whole numbers e, from a table."""
    table = torch.tensor([2.0 ** k for k in range(-300, 301)], dtype=torch.float64, device=e.device)
    return table[e.long() + 300]


def _store64(x, fmt):
    """What a row-blocked 8-bit store of x stands for, from its definition."""
    T, H = x.shape
    x = x.double()
    pad = torch.zeros(T, -H % BLOCK, dtype=x.dtype, device=x.device)
    b = torch.cat([x, pad], 1).unflatten(1, (-1, BLOCK))
    m = b.abs().max(-1, keepdim=True).values
    e = torch.frexp(m).exponent - 1
    if fmt == "int8":
        step = _power((e - 6).clamp(min=MIN_E))
        v = torch.minimum((b / step).abs().round(), torch.full_like(b, 127.0)) * b.sign() * step
    else:
        unit = _power((e - 8).clamp(min=MIN_E))
        unit = torch.where(m > 448 * unit, 2 * unit, unit)
        u = b / unit
        step = _power((torch.frexp(u).exponent - 1).clamp(min=-6) - 3)
        v = (u / step).round() * step * unit
    return v.flatten(1)[:, :H]


def _rms64(x):
    return (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()


def exact(case, seed):
    s = prepare(case, seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    d = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() and k != "codes" else v
         for k, v in s.items()}
    if kind == "store":
        return {"x": _store64(s["x"], case["fmt"])}
    if kind == "recompute8":
        unit = _power(s["exps"].int() - 127).repeat_interleave(BLOCK, 1)[:, :case["hidden"]]
        x = s["codes"].double() * unit
        h = x + d["a"]
        kept = h.to(dt).double()  # the second norm is of h as stored
        return {"y": d["w"] * x / _rms64(x), "h": h, "z": d["w2"] * kept / _rms64(kept)}
    if kind == "norm8":
        y = d["w"] * d["x"] / _rms64(d["x"])
        x = _store64(s["x"], case["fmt"])
        rms = _rms64(x)
        unit, g = x / rms, d["dy"] * d["w"]
        dx = (g - unit * ((unit * g).sum(-1, keepdim=True) / case["hidden"])) / rms
        if s["dres"] is not None:
            dx = dx + d["dres"]
        return {"y": y, "dx": dx, "dw": (d["dy"] * unit).sum(0)}
    if kind == "rotary":
        return _exact_rotary(case, d)
    return _exact_norms(case, d, dt)


def _exact_norms(case, d, dt):
    H, s = case["hidden"], case["scale"]
    g = torch.ones(1, dtype=torch.float64, device=DEV) if d["gate"] is None else d["gate"]
    unit_a, rms_a = d["a"], 1.0
    if case["post"]:
        rms_a = _rms64(d["a"])
        unit_a = d["a"] / rms_a
    w_post = d["w_post"] if case["post"] else torch.ones(H, dtype=torch.float64, device=DEV)
    h = d["x"] + s * g * (unit_a * w_post)
    out = {"h": h}
    total = d["dh"]
    if case["pre"]:
        kept = h.to(dt).double()  # the norm before the next block is of h as stored
        rms = _rms64(kept)
        unit = kept / rms
        out["y"] = unit * d["w_pre"]
        if case["way"] == "both":
            t = d["dy"] * d["w_pre"]
            total = total + (t - unit * ((t * unit).sum(-1, keepdim=True) / H)) / rms
            out["dw_pre"] = (d["dy"] * unit).sum(0)
    if case["way"] == "fwd":
        return out
    out["dx"] = total
    t = total * (s * g) * w_post
    if case["post"]:
        out["dw_post"] = ((total * (s * g)) * unit_a).sum(0)
        t = (t - unit_a * ((t * unit_a).sum(-1, keepdim=True) / H)) / rms_a
    out["da"] = t
    if case["gate"] != "none":
        per = s * total * unit_a * w_post
        out["dgate"] = per.sum(0) if case["gate"] == "channel" else per
    return out


def _exact_rotary(case, d):
    n, off, D = case["rot"] // 2, case["offset"], case["head_dim"]
    first = torch.arange(n, device=DEV) + off if case["layout"] == "half" else 2 * torch.arange(n, device=DEV) + off
    second = first + (n if case["layout"] == "half" else 1)
    phase = torch.outer(d["pos"].double(), d["inv_freq"])
    turn = torch.polar(torch.full_like(phase, d["factor"]), phase)[:, None, :]

    def apply(x, by):
        x = x.unflatten(1, (-1, D)).clone()
        z = torch.complex(x[..., first], x[..., second]) * by
        x[..., first], x[..., second] = z.real, z.imag
        return x.flatten(1)

    out = {"q": apply(d["q"], turn), "k": apply(d["k"], turn)}
    if case["way"] == "both":
        out["dq"], out["dk"] = apply(d["dq"], turn.conj()), apply(d["dk"], turn.conj())
    return out
