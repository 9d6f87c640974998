"""The operators around a checkpointed block together, as a training step and as an answer of
single tokens use them, against the same block from plain operations in fp64."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
H, HEADS, KV, HD, ROT = 256, 4, 2, 64, 32


class _Norm8(torch.autograd.Function):
    """RMSNorm in fp64 whose backward is taken at the value that 8 bits keep of x."""

    @staticmethod
    def forward(ctx, x, w, kept):
        ctx.save_for_backward(w, kept)
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w

    @staticmethod
    def backward(ctx, dy):
        w, x = ctx.saved_tensors
        r = 1 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        g, n = dy * w, x * r
        return r * (g - n * (g * n).mean(-1, keepdim=True)), (dy * n).flatten(0, -2).sum(0), None


def _weights(dtype):
    shapes = dict(w_in=(H,), wqkv=((HEADS + 2 * KV) * HD, H), wo=(H, HEADS * HD), w_post=(H,), w_pre=(H,), gate=(H,))
    return {k: ((1 + randn(s, 100 + i, 0.1)) if len(s) == 1 else randn(s, 100 + i, 0.05)).to(dtype).to(DEV).requires_grad_(True)
            for i, (k, s) in enumerate(shapes.items())}


def _attention(q, k, v):
    """Causal attention of [B, S, heads * HD] in plain products."""
    B, S, _ = q.shape
    q, k, v = (t.reshape(B, S, -1, HD).transpose(1, 2).contiguous() for t in (q, k, v))
    k, v = (t.repeat_interleave(HEADS // KV, 1).contiguous() for t in (k, v))
    s = (q @ k.transpose(-1, -2).contiguous()) / HD ** 0.5
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
    return (s.softmax(-1) @ v).transpose(1, 2).reshape(B, S, HEADS * HD)


def _block(w, x, pos, freq, factor, fmt):
    """A norm kept in 8 bits, rotary attention, the norms after and before, in fp32."""
    from transformers.models.llama.modeling_llama import LlamaRMSNorm

    from femtotron_amd import apply_rotary, block_norms, eight_bit_checkpoint
    norm = LlamaRMSNorm(H, eps=EPS).to(DEV)
    norm.weight = nn.Parameter(w["w_in"].detach())
    y = eight_bit_checkpoint(fmt)(norm, x, use_reentrant=False) if fmt else norm(x)
    qkv = y @ w["wqkv"].t()
    q, k, v = qkv.split([HEADS * HD, KV * HD, KV * HD], -1)
    q, k = apply_rotary(q, k, pos, freq, head_dim=HD, rot_dim=ROT, offset=16, layout="interleaved", factor=factor)
    a = _attention(q, k, v) @ w["wo"].t()
    h, z = block_norms(x, a, w["w_post"], w["w_pre"], gate=w["gate"], scale=0.5, eps=EPS)
    return h, z, norm.weight


def _plain(w, x, pos, freq, factor, kept):
    if kept is None:
        y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w["w_in"]
    else:
        y = _Norm8.apply(x, w["w_in"], kept)
    qkv = y @ w["wqkv"].t()
    q, k, v = qkv.split([HEADS * HD, KV * HD, KV * HD], -1)
    angle = pos.double()[:, None, None] * freq
    c, s = factor * angle.cos(), factor * angle.sin()

    def turn(t):
        t = t.unflatten(-1, (-1, HD))
        u, p = t[..., 16:16 + ROT:2], t[..., 17:16 + ROT:2]
        both = torch.stack([u * c - p * s, p * c + u * s], -1).flatten(-2)
        return torch.cat([t[..., :16], both, t[..., 16 + ROT:]], -1).flatten(-2)

    a = _attention(turn(q), turn(k), v) @ w["wo"].t()
    n = a / (a.square().mean(-1, keepdim=True) + EPS).sqrt() * w["w_post"]
    h = x + 0.5 * w["gate"] * n
    return h, h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w["w_pre"]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,S", [(2, 33), (1, 1), (3, 64)])
def test_a_training_step_of_a_block(B, S, fmt):
    """fp32 against fp64: every value passes sums of at most 512 terms, a softmax and two
    norms, each off by a few of fp32's 2^-24 times the square root of its terms; together
    under 2^-24 * 4096 of a tensor's largest entry."""
    from femtotron_amd import ops, rotary_frequencies
    freq, factor = rotary_frequencies(ROT, 1e4, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}, device=DEV)
    pos = torch.arange(S, device=DEV) + 1000
    w, x = _weights(torch.float32), randn((B, S, H), 1).to(DEV).requires_grad_(True)
    gh, gz = randn((B, S, H), 2).to(DEV), randn((B, S, H), 3).to(DEV)
    h, z, w_in = _block(w, x, pos, freq, factor, fmt)
    names = ["wqkv", "wo", "w_post", "w_pre", "gate"]
    got = [h, z, *torch.autograd.grad((h, z), [x, w_in, *(w[n] for n in names)], (gh, gz))]
    w64 = {k: v.detach().double().requires_grad_(True) for k, v in w.items()}
    x64 = x.detach().double().requires_grad_(True)
    kept = ops.unpack8(ops.pack8(x.detach(), fmt), torch.float32).double()
    h64, z64 = _plain(w64, x64, pos, freq, factor, kept)
    ref = [h64, z64, *torch.autograd.grad((h64, z64), [x64, w64["w_in"], *(w64[n] for n in names)], (gh.double(), gz.double()))]
    for name, a, b in zip(["h", "z", "dx", "dw_in", *names], got, ref):
        assert a.shape == b.shape
        a, b = a.detach(), b.detach()
        assert float((a - b).abs().max()) <= 4096 * 2.0 ** -24 * float(b.abs().max()), name


def test_an_answer_of_single_tokens_is_the_whole_sequence():
    """Without gradients, token by token with the positions each has, as the rows of one call."""
    from femtotron_amd import apply_rotary, block_norms, ops, rotary_frequencies
    freq, factor = rotary_frequencies(HD, 5e5, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}, device=DEV)
    T = 12
    pos = torch.arange(T, device=DEV) + 100000
    x, a, q, k = (randn((T, n), 10 + i).bfloat16().to(DEV) for i, n in enumerate((H, H, HEADS * HD, KV * HD)))
    w1, w2, g = ((1 + randn((H,), 20 + i, 0.1)).bfloat16().to(DEV) for i in range(3))
    how = dict(head_dim=HD, factor=factor)
    whole = (*block_norms(x, a, w1, w2, gate=g), *apply_rotary(q, k, pos, freq, **how), ops.unpack8(ops.pack8(x)))
    for t in range(T):
        r = slice(t, t + 1)
        one = (*block_norms(x[r], a[r], w1, w2, gate=g), *apply_rotary(q[r], k[r], pos[r], freq, **how),
               ops.unpack8(ops.pack8(x[r])))
        assert all(torch.equal(p[r], o) for p, o in zip(whole, one)), t


def test_two_streams_at_once():
    """The same operators on two streams without order between them, each on its own tensors."""
    from femtotron_amd import ops, rotary_frequencies
    freq, _ = rotary_frequencies(HD, device=DEV)

    def work(seed):
        x, a, dy = (randn((2000, H), seed + i).bfloat16().to(DEV) for i in range(3))
        w = (1 + randn((H,), seed + 3, 0.1)).bfloat16().to(DEV)
        pos = torch.arange(2000, device=DEV)
        r1, r2 = torch.empty(2000, device=DEV), torch.empty(2000, device=DEV)

        def run():
            y, p = ops.rmsnorm_fwd_pack8(x, w, EPS)
            h, z = ops.block_norms_fwd(x, a, w, w, EPS, gate=w, rstd_post=r1, rstd_pre=r2)
            q, _ = ops.rotary_fwd(x, None, pos, freq, head_dim=HD)
            return (y, h, z, q, *ops.rmsnorm_bwd8(dy, p, w, EPS),
                    *ops.block_norms_bwd(dy, dy, h, a, w, w, gate=w, rstd_post=r1, rstd_pre=r2))
        return run

    runs = [work(30), work(40)]
    refs = [[t.clone() for t in run()] for run in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (run, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[i].append(run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for outs in got[i] for a, b in zip(outs, refs[i]))
