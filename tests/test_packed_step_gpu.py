"""The operators of a step over packed documents together, as a training step and its answers use
them, against the same step from plain operations in fp64."""
from __future__ import annotations

import pytest
import torch

from tests import masked_reference as mr
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
V, H, HEADS, KV, HD, EPS, CAP = 300, 256, 4, 2, 64, 1e-5, 8.0


def _weights(dtype):
    shapes = dict(embed=(V, H), w_in=(H,), wqkv=((HEADS + 2 * KV) * HD, H), wo=(H, HEADS * HD), w_post=(H,), w_pre=(H,))
    return {k: ((1 + randn(s, 100 + i, 0.1)) if len(s) == 1 else randn(s, 100 + i, 0.05)).to(dtype).to(DEV).requires_grad_(True)
            for i, (k, s) in enumerate(shapes.items())}


def _norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def _own_step(w, ids, starts, lengths, positions, freq, slopes):
    from femtotron_amd import apply_rotary, attention_mask, block_norms, embedding, masked_attention
    B, S = ids.shape
    x = embedding(ids, w["embed"], factor=H ** 0.5)
    qkv = _norm(x, w["w_in"]) @ w["wqkv"].t()
    q, k, v = qkv.split([HEADS * HD, KV * HD, KV * HD], -1)
    q, k = apply_rotary(q, k, positions, freq, head_dim=HD)
    mask = attention_mask(B, S, starts, lengths)
    a = masked_attention(q, k, v, mask, head_dim=HD, cap=CAP, slopes=slopes) @ w["wo"].t()
    h, y = block_norms(x, a, w["w_post"], w["w_pre"], eps=EPS)
    return y


def _turn(t, positions, freq):
    angle = positions.double().reshape(-1, 1, 1) * freq
    c, s = angle.cos(), angle.sin()
    t = t.reshape(positions.numel(), -1, HD)
    u, p = t[..., :HD // 2], t[..., HD // 2:]
    return torch.cat([u * c - p * s, p * c + u * s], -1)


def _plain_step(w, ids, see, positions, freq, slopes):
    B, S = ids.shape
    x = w["embed"][ids] * H ** 0.5
    q, k, v = (_norm(x, w["w_in"]) @ w["wqkv"].t()).split([HEADS * HD, KV * HD, KV * HD], -1)
    q, k = (_turn(t, positions, freq).transpose(0, 1) for t in (q, k))
    v = v.reshape(B * S, KV, HD).transpose(0, 1)
    k, v = (t.repeat_interleave(HEADS // KV, 0) for t in (k, v))
    i = torch.arange(B * S, device=DEV)
    z = CAP * torch.tanh(q @ k.mT / HD ** 0.5 / CAP) - slopes.double()[:, None, None] * (i[:, None] - i).abs()
    p = torch.softmax(z.masked_fill(~see, -1e300), -1) * see
    a = (p @ v).transpose(0, 1).reshape(B, S, HEADS * HD) @ w["wo"].t()
    return _norm(x + _norm(a, w["w_post"]), w["w_pre"])


def test_a_training_step_with_clipping():
    """fp32 against fp64: values pass sums of at most 512 terms, a softmax and three norms, each off
    by a few of fp32's 2^-24 times the root of its terms; together under 2^-24 * 4096 of a
    tensor's largest entry."""
    from femtotron_amd import rotary_frequencies
    from femtotron_amd.optim import clip_grad_norm_
    B, S = 2, 70
    starts, lengths = [0, 33, 70, 100], [33, 30, 30, 40]  # padding behind both rows
    freq, _ = rotary_frequencies(HD, device=DEV)
    slopes = torch.tensor([0.3, 0.1, 0.03, 0.01], device=DEV)
    positions = torch.cat([torch.arange(33), torch.arange(37), torch.arange(30), torch.arange(40)]).to(DEV)
    ids = torch.randint(V, (B, S), generator=torch.Generator().manual_seed(5)).to(DEV)
    dy = randn((B, S, H), 6).to(DEV)
    see = mr.seen(*mr.ranges(B, S, starts, lengths), B * S, DEV)
    dy.view(B * S, H)[~see.any(-1)] = 0  # a loss leaves padding out
    w = _weights(torch.float32)
    y = _own_step(w, ids, torch.tensor(starts, device=DEV), torch.tensor(lengths, device=DEV), positions, freq, slopes)
    y.backward(dy)
    w64 = {k: t.detach().double().requires_grad_(True) for k, t in w.items()}
    y64 = _plain_step(w64, ids, see, positions, freq, slopes)
    y64.backward(dy.double())
    grads = {k: t.grad.clone() for k, t in w.items()}
    rows = see.any(-1)
    for name, a, b in [("y", y.detach().view(-1, H)[rows], y64.detach().view(-1, H)[rows])] + \
            [(k, grads[k], w64[k].grad) for k in w]:
        assert float((a - b).abs().max()) <= 4096 * 2.0 ** -24 * float(b.abs().max()), name
    norm = clip_grad_norm_(list(w.values()), 0.5)
    want = float(torch.stack([t.grad.square().sum() for t in w64.values()]).sum().sqrt())
    assert abs(float(norm) - want) <= 4096 * 2.0 ** -24 * want and want > 0.5
    for k, t in w.items():
        assert torch.equal(t.grad, grads[k] * torch.tensor(0.5 / (float(norm) + 1e-6), device=DEV)) or \
            float((t.grad - grads[k] * 0.5 / (float(norm) + 1e-6)).abs().max()) <= 2.0 ** -22 * float(t.grad.abs().max())


def test_answers_of_single_tokens_are_the_sequences():
    """Two sequences answered token by token over their caches, as one batch of causal rows."""
    from femtotron_amd import apply_rotary, attention_mask, cache_attention, embedding, masked_attention, rotary_frequencies
    B, T = 2, 20
    freq, _ = rotary_frequencies(HD, device=DEV)
    w = {k: t.detach() for k, t in _weights(torch.float32).items()}
    ids = torch.randint(V, (B, T), generator=torch.Generator().manual_seed(8)).to(DEV)
    lengths = [20, 13]

    def project(ids, positions):
        qkv = _norm(embedding(ids, w["embed"], factor=H ** 0.5), w["w_in"]) @ w["wqkv"].t()
        q, k, v = qkv.split([HEADS * HD, KV * HD, KV * HD], -1)
        return (*apply_rotary(q, k, positions, freq, head_dim=HD), v)

    q, k, v = project(ids, torch.arange(T, device=DEV))
    whole = masked_attention(q, k, v, attention_mask(B, T, lengths=torch.tensor(lengths, device=DEV)), head_dim=HD, cap=CAP)
    kc, vc = (torch.full((B, 64, KV * HD), float("nan"), device=DEV) for _ in range(2))
    for t in range(T):
        qt, kt, vt = project(ids[:, t:t + 1], torch.tensor([t], device=DEV))
        kc[:, t:t + 1], vc[:, t:t + 1] = kt, vt
        o = cache_attention(qt, kc, vc, torch.full((B,), t + 1, device=DEV), head_dim=HD, cap=CAP)
        for b in range(B):
            if t < lengths[b]:
                # fp32 sums of at most 256 terms in another order
                assert float((o[b, 0] - whole[b, t]).abs().max()) <= 2.0 ** -24 * 512 * float(whole[b].abs().max())


def test_two_streams_at_once():
    from femtotron_amd import attention_mask, cache_attention, masked_attention

    def work(seed):
        q, k, v = (randn((2000, n * HD), seed + i).bfloat16().to(DEV) for i, n in enumerate((8, 2, 2)))
        kc, vc = (t.view(4, 500, 2 * HD) for t in (k, v))
        starts = torch.tensor([0, 700, 1500], device=DEV)
        lengths = torch.tensor([500, 3, 200, 77], device=DEV)

        def run():
            o = masked_attention(q, k, v, attention_mask(1, 2000, starts), head_dim=HD, cap=20.0)
            return o, cache_attention(q[:4].view(4, 1, -1), kc, vc, lengths, head_dim=HD)
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
