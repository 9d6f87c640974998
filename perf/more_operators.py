"""The operators of a training step over packed documents, and of its answers, whose speed is
followed: their cases, their plain forms and their values in 64 bits.

* ``attend``: attention of the documents packed into the rows of a batch: each token sees its
  own document, up to itself (``see`` "causal"), all of it ("both"), or up to itself and the
  document's prefix ("prefix"); the last ``window`` tokens of it where one is set.  Scores are
  capped (cap * tanh(score / cap)) where ``cap`` is set, and ``bias`` subtracts a slope of the
  head times the distance.  Rows end in ``pad`` tokens of no document.
* ``cache``: the same scores for ``new`` tokens of each sequence over a cache of its keys and
  values; the sequences have lengths of their own.
* ``embed``: the embedding with a factor, forward alone or with its gradient.
* ``clip``: the norm of all gradients of a model and their clipping into the gradients of the
  optimizer's fp32 copies, or of the same type.

Widths are those of the repository's configurations (8 heads of 32 over 4, 32 of 64 over 4, 32
of 128 over 8 or 32; hidden 256, 2048, 4096), token counts run from one to the configured ones.
Documents' lengths are those of a case, their order in a row a seed's.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}

# hidden, query heads, kv heads, head_dim, ffn, vocabulary
WIDTHS = {
    "debug": (256, 8, 4, 32, 688, 1024),
    "tinyllama": (2048, 32, 4, 64, 5632, 32000),
    "llama3-8b": (4096, 32, 8, 128, 14336, 128256),
    "llama2-7b": (4096, 32, 32, 128, 11008, 32000),
}


# ------------------------------------------------------------------ cases
def _attend(width, batch, seq, dtype="bf16", way="both", see="causal", docs=0, pad=0, window=0, cap=0.0, bias=False):
    _, heads, kv, head_dim, _, _ = WIDTHS[width]
    return dict(kind="attend", way=way, batch=batch, seq=seq, heads=heads, kv=kv, head_dim=head_dim, see=see, docs=docs,
                pad=pad, window=window, cap=cap, bias=bias, dtype=dtype)


def _cache(width, batch, room, new=1, dtype="bf16", window=0, cap=0.0, bias=False):
    _, heads, kv, head_dim, _, _ = WIDTHS[width]
    return dict(kind="cache", batch=batch, room=room, new=new, heads=heads, kv=kv, head_dim=head_dim, window=window,
                cap=cap, bias=bias, dtype=dtype)


def _embed(width, tokens, dtype="bf16", way="both", ids="zipf"):
    hidden, _, _, _, _, vocab = WIDTHS[width]
    return dict(kind="embed", way=way, tokens=tokens, hidden=hidden, vocab=vocab, ids=ids, dtype=dtype)


def _clip(width, layers, dtype="bf16", into="fp32"):
    return dict(kind="clip", width=width, layers=layers, dtype=dtype, into=into)


def listed():
    return [
        # The fp32 debug model's batch, each row's first tokens a prompt that all of it sees: launches are the time.
        dict(name="attend_debug_fp32", **_attend("debug", 2, 128, "fp32", see="prefix")),
        # A ragged batch of padded rows whose scores fall with the distance.
        dict(name="attend_ragged", **_attend("tinyllama", 3, 333, docs=90, pad=21, bias=True)),
        # The configured TinyLlama training step's attention with documents packed into its rows.
        dict(name="attend_train", **_attend("tinyllama", 8, 2048, docs=600)),
        # The 8B width at its configured 8192 tokens, one long document, scores capped.
        dict(name="attend_8b", **_attend("llama3-8b", 1, 8192, cap=50.0)),
        # One token of one sequence while answering: launches are the time.
        dict(name="cache_token", **_cache("tinyllama", 1, 2048)),
        # A batch of answers, scores capped as in training.
        dict(name="cache_batch", **_cache("llama3-8b", 32, 8192, cap=50.0)),
        # A few new tokens of each of a few long sequences, scores falling with the distance.
        dict(name="cache_long", **_cache("llama2-7b", 2, 32768, new=5, bias=True)),
        # A few tokens while answering.
        dict(name="embed_token", **_embed("llama3-8b", 4, way="fwd")),
        # The training step's tokens, text-like ids.
        dict(name="embed_train", **_embed("tinyllama", 16384)),
        # A large vocabulary of which a step meets little.
        dict(name="embed_8b", **_embed("llama3-8b", 8192)),
        # The debug model's gradients: launches are the time.
        dict(name="clip_debug", **_clip("debug", 2, "fp32")),
        # All gradients of the TinyLlama model, bf16 into the optimizer's fp32.
        dict(name="clip_tinyllama", **_clip("tinyllama", 22)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "cache", "cache", "embed", "clip"])
    width = rng.choice(["debug", "tinyllama", "tinyllama", "llama3-8b", "llama2-7b"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    score = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.choice([False, False, True]))
    if kind == "attend":
        batch, way = rng.choice([1, 1, 2, 3, 8]), rng.choice(["fwd", "both", "both"])
        most = 1024 if dtype == "fp32" else 5800 if WIDTHS[width][3] < 128 else 4096
        # a token that sees itself alone has no gradient in q and k: such rows are few in a training case
        least = 1 if way == "fwd" else 8
        seq = _log(rng, least, most // batch)
        see = rng.choice(["causal", "causal", "both", "prefix"])
        window = _log(rng, least, 2 * seq) if see != "prefix" and rng.random() < 0.3 else 0
        return _attend(width, batch, seq, dtype, way=way, see=see, window=window,
                       docs=rng.choice([0, _log(rng, 2 * least - 1, 2 * seq)]), pad=rng.choice([0, rng.randrange((seq + 1) // 2)]), **score)
    if kind == "cache":
        batch = rng.choice([1, 2, 5, 16, 32])
        most = (1 << 28) // (batch * WIDTHS[width][2] * WIDTHS[width][3] * (2 if dtype == "fp32" else 1))
        room = _log(rng, 1, min(32768, most))
        return _cache(width, batch, room, rng.choice([1, 1, 1, 2, 5, 16]), dtype, rng.choice([0, 0, _log(rng, 1, room)]), **score)
    if kind == "embed":
        if dtype == "fp32" and width == "llama3-8b":
            width = "tinyllama"
        return _embed(width, _log(rng, 1, 16384), dtype, rng.choice(["fwd", "both", "both"]), rng.choice(["zipf", "uniform"]))
    if width == "llama3-8b":
        width = "llama2-7b"
    layers = 3 if width == "llama2-7b" else 22
    return _clip(width, rng.randint(1, layers // 2 if dtype == "fp32" else layers), dtype, rng.choice(["fp32", "same"]))


# ------------------------------------------------------------------ inputs
def _documents(case):
    """The lengths of a row's documents: a spread of four to one and more around the mean."""
    left, mean = case["seq"] - case["pad"], case["docs"]
    if not mean:
        return [left]
    rng, lengths = random.Random(7), []
    while left:
        n = min(left, max(1, int(mean * math.exp(rng.gauss(-0.2, 0.6)))))
        lengths.append(n)
        left -= n
    return lengths


def _prefix(length):
    return length // 3


def _lengths(case):
    """The lengths of a cache's sequences: from full to an eighth of its room."""
    rng, room = random.Random(11), case["room"]
    return [room if i == 0 else max(1, int(room * 8 ** -rng.random())) for i in range(case["batch"])]


def _slopes(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _gradients(case):
    """The shapes of a model's gradients."""
    hidden, heads, kv, head_dim, ffn, vocab = WIDTHS[case["width"]]
    layer = [(heads * head_dim, hidden), (kv * head_dim, hidden), (kv * head_dim, hidden), (hidden, heads * head_dim),
             (ffn, hidden), (ffn, hidden), (hidden, ffn), (hidden,), (hidden,)]
    return [(vocab, hidden)] + layer * case["layers"] + [(hidden,), (vocab, hidden)]


def _normal(gen, *shape, dtype, std=1.0):
    return torch.randn(*shape, generator=gen, device=DEV).mul_(std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = random.Random(int(seed))
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    s = dict(case=case)
    if kind in ("attend", "cache"):
        wq, wk = case["heads"] * case["head_dim"], case["kv"] * case["head_dim"]
        # capped models' scores are large
        std = 3.0 if case["cap"] else 1.0
        s["slopes"] = torch.tensor(_slopes(case["heads"]), device=DEV) if case["bias"] else None
    if kind == "attend":
        B, S = case["batch"], case["seq"]
        qkv = _normal(gen, B, S, wq + 2 * wk, dtype=dt)  # q, k and v are columns of the packed projection
        qkv[..., :wq].mul_(std)
        s["q"], s["k"], s["v"] = qkv[..., :wq], qkv[..., wq:wq + wk], qkv[..., wq + wk:]
        s["do"] = _normal(gen, B, S, wq, dtype=dt, std=0.01)
        starts, lengths = [], []
        for b in range(B):
            row = _documents(case)
            rng.shuffle(row)
            at = b * S
            for n in row:
                starts.append(at)
                lengths.append(n)
                at += n
        s["starts"] = torch.tensor(starts, device=DEV)
        s["lengths"] = torch.tensor(lengths, device=DEV)
        s["prefix"] = torch.tensor([_prefix(n) for n in lengths], device=DEV) if case["see"] == "prefix" else None
        if case["way"] == "both":
            for k in ("q", "k", "v"):
                s[k].requires_grad_(True)
    elif kind == "cache":
        lengths = _lengths(case)
        rng.shuffle(lengths)
        s["lengths"] = torch.tensor(lengths, device=DEV)
        s["q"] = _normal(gen, case["batch"], case["new"], wq, dtype=dt, std=std)
        s["k"] = _normal(gen, case["batch"], case["room"], wk, dtype=dt)
        s["v"] = _normal(gen, case["batch"], case["room"], wk, dtype=dt)
    elif kind == "embed":
        T, V, H = case["tokens"], case["vocab"], case["hidden"]
        if case["ids"] == "uniform":
            s["ids"] = torch.randint(V, (T,), generator=gen, device=DEV)
        else:  # frequency falls as one over the rank; ranks are spread over the vocabulary
            u = torch.rand(T, generator=gen, device=DEV, dtype=torch.float64)
            rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
            s["ids"] = rank * 7919 % V
        s["factor"] = math.sqrt(H)
        s["w"] = _normal(gen, V, H, dtype=dt, std=0.02)
        s["dy"] = _normal(gen, T, H, dtype=dt, std=0.01)
        if case["way"] == "both":
            s["w"].requires_grad_(True)
    else:
        s["grads"] = [_normal(gen, *shape, dtype=dt, std=0.01 * math.exp(rng.gauss(0, 0.5))) for shape in _gradients(case)]
        into = torch.float32 if case["into"] == "fp32" else dt
        # the optimizer's gradients lie in one buffer
        s["out"] = torch.empty(sum(g.numel() for g in s["grads"]), dtype=into, device=DEV)
        at, s["views"] = 0, []
        for g in s["grads"]:
            s["views"].append(s["out"][at:at + g.numel()].view(g.shape))
            at += g.numel()
        s["max_norm"] = 1.0
    return s


# ------------------------------------------------------------------ plain forms
def _seen(s):
    """[batch, seq, seq]: whether row i of a batch's row sees row j."""
    c = s["case"]
    B, S = c["batch"], c["seq"]
    row = torch.arange(B * S, device=DEV)
    starts, ends = s["starts"], s["starts"] + s["lengths"]
    doc = (starts <= row[:, None]).sum(1) - 1
    begin, end = starts[doc], ends[doc]
    lo, hi = begin, row + 1
    if c["see"] == "both":
        hi = end
    elif c["see"] == "prefix":
        hi = torch.maximum(hi, begin + s["prefix"][doc])
    if c["window"]:
        lo = torch.maximum(lo, row + 1 - c["window"])
        hi = torch.minimum(hi, row + c["window"])
    hi = torch.where(row < end, hi, lo)
    j = row.view(B, 1, S)
    return (lo.view(B, S, 1) <= j) & (j < hi.view(B, S, 1))


def _split(x, kv, group, head_dim):
    """[B, n, heads * head_dim] as [B * kv, group * n, head_dim] in fp32."""
    B, n, _ = x.shape
    return x.detach().float().view(B, n, kv, group, head_dim).permute(0, 2, 3, 1, 4).reshape(B * kv, group * n, head_dim)


def _join(x, B, kv, group, dtype):
    """_split's inverse, rounded."""
    n = x.shape[1] // group
    return x.view(B, kv, group, n, -1).permute(0, 3, 1, 2, 4).reshape(B, n, -1).to(dtype)


def _weights(s, q, k, seen, distance):
    """The softmax weights [B * kv, group, n, keys] of split q and k, and tanh of the capped scores."""
    c = s["case"]
    kv, group = c["kv"], c["heads"] // c["kv"]
    z = (q * c["head_dim"] ** -0.5) @ k.transpose(1, 2).contiguous()
    t = None
    if c["cap"]:
        t = (z / c["cap"]).tanh_()
        z = t * c["cap"]
    z = z.view(-1, kv, group, *seen.shape[1:])
    if c["bias"]:
        z = z - s["slopes"].view(1, kv, group, 1, 1) * distance[:, None, None]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    z = (z - z.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = z.sum(-1, keepdim=True)
    p = z.div_(total.masked_fill_(total == 0, 1.0))
    return p.view(q.shape[0], q.shape[1], -1), t


def _plain_attend(s):
    c = s["case"]
    B, S, kv, group, D = c["batch"], c["seq"], c["kv"], c["heads"] // c["kv"], c["head_dim"]
    dt, scale = s["q"].dtype, c["head_dim"] ** -0.5
    q, k, v = _split(s["q"], kv, group, D), _split(s["k"], kv, 1, D), _split(s["v"], kv, 1, D)
    i = torch.arange(S, device=DEV)
    p, t = _weights(s, q, k, _seen(s), (i[:, None] - i).abs()[None])
    o = p @ v
    out = {"o": _join(o, B, kv, group, dt)}
    if c["way"] == "both":
        do = _split(s["do"], kv, group, D)
        out["dv"] = _join(p.transpose(1, 2).contiguous() @ do, B, kv, 1, dt)
        dz = do @ v.transpose(1, 2).contiguous()
        dz = dz.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
        if t is not None:
            dz = dz.mul_(1 - t.square_())
        out["dq"] = _join(scale * (dz @ k), B, kv, group, dt)
        out["dk"] = _join(scale * (dz.transpose(1, 2).contiguous() @ q), B, kv, 1, dt)
    return out


def _cache_seen(s):
    c = s["case"]
    at = s["lengths"][:, None] - c["new"] + torch.arange(c["new"], device=DEV)  # the new tokens' places
    j = torch.arange(c["room"], device=DEV)
    away = at[:, :, None] - j
    seen = away >= 0
    if c["window"]:
        seen = seen & (away < c["window"])
    return seen, away


def _plain_cache(s):
    c = s["case"]
    B, kv, group, D = c["batch"], c["kv"], c["heads"] // c["kv"], c["head_dim"]
    q, k, v = _split(s["q"], kv, group, D), _split(s["k"], kv, 1, D), _split(s["v"], kv, 1, D)
    p, _ = _weights(s, q, k, *_cache_seen(s))
    return {"o": _join(p @ v, B, kv, group, s["q"].dtype)}


def _plain_embed(s):
    w, ids = s["w"].detach(), s["ids"]
    out = {"y": (w[ids].float() * s["factor"]).to(w.dtype)}
    if s["case"]["way"] == "both":
        dw = torch.zeros(w.shape, device=DEV).index_add_(0, ids, s["dy"].float())
        out["dw"] = dw.mul_(s["factor"]).to(w.dtype)
    return out


def _plain_clip(s):
    squares = torch.stack([g.double().square().sum() for g in s["grads"]])
    norm = squares.sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp_max(1.0).float()
    s["out"].copy_(torch.cat([g.view(-1) for g in s["grads"]]).float().mul_(factor))
    return {"norm": norm.float(), "grads": s["out"]}


def _plain(s):
    return {"attend": _plain_attend, "cache": _plain_cache, "embed": _plain_embed, "clip": _plain_clip}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from femtotron_amd import attention_mask, cache_attention, embedding, masked_attention
    from femtotron_amd.optim import clip_gradients
    c = s["case"]
    kind = c["kind"]
    if kind == "clip":
        return {"norm": clip_gradients(s["grads"], s["max_norm"], out=s["views"]), "grads": s["out"]}
    if kind == "embed":
        y = embedding(s["ids"], s["w"], factor=s["factor"])
        out = {"y": y.detach()}
        if c["way"] == "both":
            out["dw"], = torch.autograd.grad(y, s["w"], s["dy"])
        return out
    how = dict(head_dim=c["head_dim"], cap=c["cap"] or None, slopes=s["slopes"])
    if kind == "cache":
        return {"o": cache_attention(s["q"], s["k"], s["v"], s["lengths"], window=c["window"] or None, **how)}
    mask = attention_mask(c["batch"], c["seq"], s["starts"], s["lengths"], prefix=s["prefix"], causal=c["see"] != "both",
                          window=c["window"] or None)
    o = masked_attention(s["q"], s["k"], s["v"], mask, **how)
    out = {"o": o.detach()}
    if c["way"] == "both":
        out["dq"], out["dk"], out["dv"] = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work
def _pairs(case):
    """The (token, token) pairs of one head that are seen."""
    total = 0
    for n in _documents(case):
        w = min(case["window"] or n, n)
        behind = w * (w + 1) // 2 + (n - w) * w  # up to itself
        if case["see"] == "both":
            total += 2 * behind - n
        elif case["see"] == "prefix":
            m = _prefix(n)
            total += behind + m * (m - 1) // 2
        else:
            total += behind
    return total * case["batch"]


def work(case):
    """Each call of a pass reads its inputs and writes its outputs once: a backward is a call of
    its own, later, and reads again what the forward had and gave (o, and a value a row and head)."""
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "attend":
        rows, heads, kv, D = case["batch"] * case["seq"], case["heads"], case["kv"], case["head_dim"]
        q, k, stats = rows * heads * D * size, rows * kv * D * size, rows * heads * 4
        both = case["way"] == "both"
        return {"bytes": 2 * q + 2 * k + (4 * q + 4 * k + 2 * stats if both else 0),
                "flops": _pairs(case) * heads * D * (14 if both else 4)}
    if kind == "cache":
        heads, kv, D = case["heads"], case["kv"], case["head_dim"]
        reach = (case["window"] + case["new"] - 1) if case["window"] else case["room"]
        rows = sum(min(n, reach) for n in _lengths(case))
        return {"bytes": (2 * rows * kv + 2 * case["batch"] * case["new"] * heads) * D * size,
                "flops": 4 * rows * case["new"] * heads * D}
    if kind == "embed":
        rows = case["tokens"] * case["hidden"] * size
        if case["way"] == "fwd":
            return {"bytes": 2 * rows + 8 * case["tokens"], "flops": rows // size}
        return {"bytes": 3 * rows + 16 * case["tokens"] + case["vocab"] * case["hidden"] * size, "flops": 3 * rows // size}
    n = sum(math.prod(shape) for shape in _gradients(case))
    return {"bytes": n * (size + (4 if case["into"] == "fp32" else size)), "flops": 3 * n}


# ------------------------------------------------------------------ values in 64 bits
def _softmax64(z, seen):
    """Rows of weights; zeros in a row that sees nothing."""
    w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
    return torch.where(seen.any(-1, keepdim=True), w, 0.0)


def _scores64(case, q, k, away):
    """The scores [kv, group, n, m] of q [kv, group, n, D] and k [kv, m, D]; away [n, m]: the distances."""
    z = torch.matmul(q, k[:, None].mT) / math.sqrt(case["head_dim"])
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    if case["bias"]:
        z = z - torch.tensor(_slopes(case["heads"]), dtype=torch.float64, device=DEV).view(z.shape[0], -1, 1, 1) * away.abs()
    return z


def _heads64(x, D):
    """[n, heads * D] as [heads, n, D] in fp64."""
    return x.detach().double().unflatten(-1, (-1, D)).transpose(0, 1)


def _exact_attend(case, s):
    B, S, D, kv = case["batch"], case["seq"], case["head_dim"], case["kv"]
    group = case["heads"] // kv
    names = ("q", "k", "v", "do")
    rows = {n: _heads64(s[n].detach().reshape(B * S, -1), D) for n in names}
    out = {n: torch.zeros_like(rows[n[-1] if n != "o" else "q"]) for n in ("o", "dq", "dk", "dv")}
    prefix = s["prefix"].tolist() if s["prefix"] is not None else None
    for d, (at, n) in enumerate(zip(s["starts"].tolist(), s["lengths"].tolist())):
        i = torch.arange(n, device=DEV)
        away = i[:, None] - i
        seen = torch.ones_like(away, dtype=torch.bool) if case["see"] == "both" else away >= 0
        if prefix:
            seen |= (i < prefix[d])
        if case["window"]:
            seen &= away.abs() < case["window"]
        step = max(1, min(kv, (1 << 28) // max(1, n * n * group)))  # kv heads at a time
        for h in range(0, kv, step):
            e = min(kv, h + step)
            q = rows["q"][h * group:e * group, at:at + n].unflatten(0, (e - h, group)).requires_grad_(True)
            k, v = (rows[x][h:e, at:at + n].clone().requires_grad_(True) for x in "kv")
            o = torch.matmul(_softmax64(_scores64(case, q, k, away), seen), v[:, None])
            out["o"][h * group:e * group, at:at + n] = o.detach().flatten(0, 1)
            if case["way"] == "both":
                g = torch.autograd.grad(o, (q, k, v), rows["do"][h * group:e * group, at:at + n].unflatten(0, (e - h, group)))
                out["dq"][h * group:e * group, at:at + n] = g[0].flatten(0, 1)
                out["dk"][h:e, at:at + n], out["dv"][h:e, at:at + n] = g[1], g[2]
    keep = ("o", "dq", "dk", "dv") if case["way"] == "both" else ("o",)
    return {n: out[n].transpose(0, 1).reshape(B, S, -1) for n in keep}


def _exact_cache(case, s):
    B, n, D, kv = case["batch"], case["new"], case["head_dim"], case["kv"]
    out = []
    for b, length in enumerate(s["lengths"].tolist()):
        q = _heads64(s["q"][b], D).unflatten(0, (kv, -1))
        k, v = _heads64(s["k"][b, :length], D), _heads64(s["v"][b, :length], D)
        away = torch.arange(length - n, length, device=DEV)[:, None] - torch.arange(length, device=DEV)
        seen = away >= 0
        if case["window"]:
            seen &= away < case["window"]
        o = torch.matmul(_softmax64(_scores64(case, q, k, away), seen), v[:, None])
        out.append(o.flatten(0, 1).transpose(0, 1).reshape(n, -1))
    return {"o": torch.stack(out)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(case, s)
    if kind == "cache":
        return _exact_cache(case, s)
    if kind == "embed":
        w = s["w"].detach().double()
        out = {"y": w.index_select(0, s["ids"]) * s["factor"]}
        if case["way"] == "both":
            dw = torch.zeros_like(w).index_put_((s["ids"],), s["dy"].double(), accumulate=True)
            out["dw"] = dw * s["factor"]
        return out
    flat = torch.cat([g.flatten() for g in s["grads"]]).double()
    norm = torch.linalg.vector_norm(flat)
    return {"norm": norm, "grads": flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
