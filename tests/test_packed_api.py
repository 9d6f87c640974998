"""The operators of a step over packed documents, without a GPU: the header and its binding, refusals
on the host, derivatives and tracing that are refused, the module's CPU path."""
from __future__ import annotations

import ctypes
import hashlib
import re

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from tests import masked_reference as mr
from tests.conftest import ROOT
from tests.helpers import randn


def _header() -> str:
    return re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "femtohip_packed.h").read_text(), flags=re.S)


def _lib():
    from femtotron_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfemtohip.so not built")
    return _lib


def test_library_exports_every_symbol_of_the_packed_header():
    lib = _lib()
    declared = set(re.findall(r"\b(fh_[a-z0-9_]+)\s*\(", _header()))
    assert declared and declared == set(lib.PACKED_SIGNATURES), declared ^ set(lib.PACKED_SIGNATURES)
    raw = ctypes.CDLL(str(lib.LIB_PATH))
    for name in declared:
        assert hasattr(raw, name), name
    assert lib.lib().fh_packed_abi_version() == lib.PACKED_ABI_VERSION


# As ABI_DECLARATIONS of test_api.py: the declarations of a version of this header.
PACKED_DECLARATIONS = (1, "bbfcbcb7c162ebb3")


def test_packed_version_is_raised_with_the_declarations():
    from femtotron_amd import _lib
    text = _header()
    version = int(re.search(r"#define FH_PACKED_ABI_VERSION (\d+)", text).group(1))
    text = re.sub(r"#define FH_PACKED_ABI_VERSION \d+", "", text)
    digest = hashlib.sha256(re.sub(r"\s+", "", text).encode()).hexdigest()[:16]
    assert (version, digest) == PACKED_DECLARATIONS, "declarations changed: raise FH_PACKED_ABI_VERSION and record both"
    assert _lib.PACKED_ABI_VERSION == version


def test_a_library_without_the_packed_operators_is_refused(tmp_path, monkeypatch):
    import subprocess

    lib = _lib()
    src = tmp_path / "old.c"
    src.write_text("int fh_abi_version(void) { return %d; }\nint fh_blocks_abi_version(void) { return %d; }\n"
                   % (lib.ABI_VERSION, lib.BLOCKS_ABI_VERSION))
    so = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    monkeypatch.setattr(lib, "LIB_PATH", so)
    monkeypatch.setattr(lib, "_lib", None)
    with pytest.raises(lib.FemtoHipError, match="packed ABI 0.*rebuild"):
        lib.lib()


def test_entry_points_validate_on_the_host():
    lib = _lib()
    L = lib.lib()
    BIG = 1 << 40

    def refused(status, what):
        assert status == 1 and what in L.fh_last_error(), (status, L.fh_last_error())

    assert L.fh_attn_mask_size(0) == 0 and L.fh_attn_mask_size(-1) == 0 and L.fh_attn_mask_size(33) == (33 + 4) * 16
    assert L.fh_attn_mask(None, None, None, 0, 0, 5, 0, 1, None, None) == 0  # no tokens
    refused(L.fh_attn_mask(None, None, None, 2, 10, 4, 0, 1, 16, None), b"seq_len")
    refused(L.fh_attn_mask(None, None, None, 1, BIG, BIG, 0, 1, 16, None), b"tokens")
    refused(L.fh_attn_mask(None, None, None, 1 << 31, 1 << 30, 1 << 62, 0, 1, 16, None), b"seq_len")
    refused(L.fh_attn_mask(16, None, 16, 1, 10, 10, 3, 1, 16, None), b"prefix")
    refused(L.fh_attn_mask(16, None, 16, 1, 10, 10, 0, 0, 16, None), b"prefix")
    refused(L.fh_attn_mask(16, None, None, 1, 10, 10, -1, 1, 16, None), b"window")
    refused(L.fh_attn_mask(16, None, None, 1, 10, 10, 0, 1, 8, None), b"aligned")

    def fwd_(dt=0, q=16, ldq=128, ldk=64, T=10, nh=2, nkv=1, hd=64, scale=1.0, cap=0.0, low=None):
        return L.fh_masked_attn_fwd(dt, q, ldq, 16, ldk, 16, ldk, 16, ldq, None, low, 16, T, nh, nkv, hd, scale, cap, None, None)

    refused(fwd_(dt=7), b"dtype")
    refused(fwd_(nh=3, nkv=2), b"n_heads")
    refused(fwd_(hd=48), b"head_dim")
    refused(fwd_(ldq=120), b"q row stride")
    refused(fwd_(ldk=65), b"k row stride")
    refused(fwd_(ldq=1 << 24), b"row stride")
    refused(fwd_(scale=0.0), b"scale")
    refused(fwd_(scale=float("nan")), b"scale")
    refused(fwd_(cap=-1.0), b"cap")
    refused(fwd_(cap=float("inf")), b"cap")
    refused(fwd_(cap=4097.0), b"cap")
    refused(fwd_(cap=1e-30, scale=1.0), b"cap")
    refused(fwd_(scale=2.0 ** 61), b"scale")
    refused(fwd_(q=None), b"null")
    refused(fwd_(q=8), b"aligned")
    refused(fwd_(dt=1, low=16), b"o_low")
    assert fwd_(T=0) == 0
    assert L.fh_masked_attn_bwd_workspace_size(0, 0, 2, 1, 64) == 0
    assert L.fh_masked_attn_bwd_workspace_size(1, 100, 2, 1, 64) == 2 * 100 * 2 * 4
    # few tokens: a kv head's query heads are split, and their sums need room
    assert L.fh_masked_attn_bwd_workspace_size(0, 100, 8, 1, 64) > 2 * 100 * 8 * 4

    def cache(n_new=1, room=100, krow=64, kb=6400, window=0, batch=2, ws=16, q=16):
        return L.fh_cache_attn(0, q, 128, 16, kb, krow, 64, 16, kb, krow, 64, 16, 128, 16, batch, n_new, room, 2, 1, 64, window,
                               1.0, 0.0, None, ws, None)

    refused(cache(n_new=-1), b"negative")
    refused(cache(room=BIG), b"room")
    refused(cache(krow=63), b"k row stride")
    refused(cache(kb=6401), b"multiples of 8")
    refused(cache(kb=-6400), b"multiples of 8")
    refused(cache(window=-1), b"window")
    refused(cache(q=None), b"null")
    refused(cache(room=5000, ws=None), b"workspace")
    assert cache(batch=0) == 0 and cache(n_new=0) == 0
    assert L.fh_cache_attn_workspace_size(0, 2, 1, 100, 2, 1, 64) == 0  # a workgroup a sequence: nothing to join
    assert L.fh_cache_attn_workspace_size(0, 2, 1, 5000, 2, 1, 64) > 0
    assert L.fh_cache_attn_workspace_size(0, 4096, 1, 5000, 2, 1, 64) == 0  # sequences enough for the chip

    refused(L.fh_embedding_scaled_fwd(0, 16, 16, 16, 1, 10, 64, float("inf"), None), b"factor")
    refused(L.fh_embedding_scaled_bwd(0, 16, 16, 16, 1, 10, 64, -1, float("nan"), 16, None), b"factor")
    refused(L.fh_embedding_scaled_fwd(0, 16, 16, 16, 1, 10, 60, 2.0, None), b"hidden")

    def clip(*grads, max_norm=1.0, norm=16, ws=16):
        table = (lib.FhGrad * len(grads))(*grads)
        return L.fh_clip_grads(len(grads), ctypes.addressof(table), max_norm, norm, ws, None)

    G = lib.FhGrad
    refused(clip(G(1 << 20, 1 << 20, 100, 0, 0), G((1 << 20) + 100, (1 << 20) + 100, 100, 0, 0)), b"overlaps")
    refused(clip(G(1 << 20, 1 << 20, 100, 0, 0), G(1 << 20, 1 << 20, 100, 0, 0)), b"overlaps")
    refused(clip(G(1 << 20, 1 << 20, 100, 0, 1)), b"overlaps")                       # in place in a wider type
    refused(clip(G(1 << 20, 1 << 21, 100, 0, 1), G(1 << 21, 1 << 22, 100, 0, 1)), b"overlaps")
    refused(clip(G(1 << 20, None, 100, 0, 0), G(1 << 21, 1 << 21, 100, 0, 0)), b"null")
    refused(clip(G(None, None, 100, 0, 0)), b"null")
    refused(clip(G(1 << 20, 1 << 20, 100, 2, 2)), b"dtypes")
    refused(clip(G(1 << 20, 1 << 20, -1, 0, 0)), b"numel")
    refused(clip(G((1 << 20) + 1, (1 << 20) + 1, 5, 0, 0)), b"aligned")
    refused(clip(max_norm=-1.0), b"max_norm")
    refused(clip(max_norm=float("nan")), b"max_norm")
    refused(clip(norm=None), b"null")


# ------------------------------------------------------- calls that end before a kernel
@pytest.fixture
def no_kernel(monkeypatch):
    """Everything up to the entry point, which counts its calls; tensors on the CPU."""
    from femtotron_amd import _lib, ops
    calls = []

    class Lib:
        def __getattr__(self, name):
            if name == "fh_attn_mask_size":
                return lambda T: 16 * (T + 2 * -(-T // 32))
            return lambda *a: 64 if name.endswith("_workspace_size") else calls.append(name) or 0

    monkeypatch.setattr(ops, "_alike", lambda *a: None)
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    return calls


def _mask(T):
    from femtotron_amd import AttentionMask
    return AttentionMask(torch.empty(16 * (T + 2 * -(-T // 32)), dtype=torch.uint8), 1, T)


def _calls():
    from femtotron_amd import cache_attention, embedding, masked_attention
    q, k = torch.randn(4, 128), torch.randn(4, 64)
    w, ids, n = torch.randn(10, 64), torch.arange(4), torch.tensor([3])
    return {
        "masked q": lambda t: masked_attention(t(q), k, k, _mask(4), head_dim=64),
        "masked k": lambda t: masked_attention(q, t(k), k, _mask(4), head_dim=64),
        "masked v": lambda t: masked_attention(q, k, t(k), _mask(4), head_dim=64),
        "embedding": lambda t: embedding(ids, t(w), factor=2.0),
        "cache q": lambda t: cache_attention(t(q[:1, None]), k[None], k[None], n, head_dim=64),
        "cache v": lambda t: cache_attention(q[:1, None], k[None], t(k[None]), n, head_dim=64),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_forward_mode_derivatives_are_refused(name, no_kernel):
    call = _calls()[name]
    call(lambda t: t)
    for grad in (True, False):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises((NotImplementedError, TypeError)):
                call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
            call(lambda t: t)


@pytest.mark.parametrize("name", list(_calls()))
def test_tracing_is_refused(name, no_kernel):
    call = _calls()[name]
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(lambda x: call(lambda t: t + x))(torch.zeros(()))


def test_constants_that_want_a_gradient_are_refused(no_kernel):
    from femtotron_amd import cache_attention, embedding, masked_attention
    q, k = torch.randn(4, 128), torch.randn(4, 64)
    one = torch.ones(2, requires_grad=True)
    with pytest.raises(TypeError, match="slopes"):
        masked_attention(q, k, k, _mask(4), head_dim=64, slopes=one)
    with pytest.raises(TypeError, match="cap"):
        masked_attention(q, k, k, _mask(4), head_dim=64, cap=torch.tensor(3.0, requires_grad=True))
    with pytest.raises(TypeError, match="slopes"):
        cache_attention(q[:1, None], k[None], k[None], torch.tensor([3]), head_dim=64, slopes=one)
    with pytest.raises(TypeError, match="factor"):
        embedding(torch.arange(4), q, factor=torch.tensor(3.0, requires_grad=True))


def test_operators_refuse_the_cpu():
    from femtotron_amd import attention_mask, cache_attention, embedding, masked_attention
    from femtotron_amd.optim import clip_gradients
    _lib()
    q = torch.randn(1, 4, 128)
    for call in (lambda: attention_mask(1, 4, device="cpu"), lambda: attention_mask(1, 4, torch.zeros(1, dtype=torch.int64)),
                 lambda: masked_attention(q, q, q, _mask(4), head_dim=64),
                 lambda: cache_attention(q, q, q, torch.tensor([3]), head_dim=64),
                 lambda: embedding(torch.arange(4), q[0], factor=2.0), lambda: clip_gradients([q], 1.0)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_the_embedding_modules_cpu_path_has_the_factor():
    from femtotron_amd.boundary_ops import FusedEmbedding
    w = torch.nn.Parameter(randn((10, 16), 1))
    ids = torch.tensor([3, -1, 10, 0])
    y = FusedEmbedding(w, factor=3.0)(ids)
    assert torch.equal(y[0], 3 * w[3]) and torch.equal(y[3], 3 * w[0]) and not y[1:3].any()
    y.sum().backward()
    assert float(w.grad.sum()) == 2 * 16 * 3.0
    old = FusedEmbedding(w)
    del old.__dict__["factor"]  # as a module pickled before it had one
    assert torch.equal(old(ids)[0], w[3])


@pytest.mark.parametrize("padding_idx", [-1, 10, -11])
def test_an_embeddings_padding_idx_is_an_id(padding_idx):
    """Python's negative index would be taken for no padding."""
    from femtotron_amd import embedding
    with pytest.raises(ValueError, match="padding_idx"):
        embedding(torch.tensor([3]), torch.zeros(10, 16), padding_idx=padding_idx)


def test_no_embedding_is_left_without_the_factor():
    """An embedding that is not swapped, or has another factor already, would answer unscaled."""
    from femtotron_amd.boundary_ops import FusedEmbedding, fuse_boundary_ops
    for emb in (torch.nn.Embedding(10, 16, max_norm=1.0), torch.nn.Embedding(10, 16, sparse=True),
                FusedEmbedding(torch.nn.Parameter(torch.zeros(10, 16))), torch.nn.Identity()):
        model = torch.nn.Module()
        model.embed_tokens = emb
        with pytest.raises(ValueError, match="factor"):
            fuse_boundary_ops(model, embedding_factor=4.0)
        assert model.embed_tokens is emb and fuse_boundary_ops(model) == 0
    model.embed_tokens = torch.nn.Embedding(10, 16)
    assert fuse_boundary_ops(model, embedding_factor=4.0) == 1 and model.embed_tokens.factor == 4.0
    assert fuse_boundary_ops(model, embedding_factor=4.0) == 0  # as it is


# --------------------------------------------------------------------- the oracle
def test_the_oracle_is_softmax_attention():
    """Against torch's own fp64 attention and its gradients, where the mask is one that it has."""
    T, nh, hd = 40, 2, 32
    q, k, v, do = (randn((T, nh * hd), i).double() for i in range(4))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    lo, hi = mr.ranges(1, T, starts=[0, 17], lengths=[17, 23])
    see = mr.seen(lo, hi, T, "cpu")
    h = [t.unflatten(1, (nh, hd)).transpose(0, 1) for t in (q, k, v)]
    ref = torch.nn.functional.scaled_dot_product_attention(*h, attn_mask=see).transpose(0, 1).flatten(1)
    g = torch.autograd.grad(ref, (q, k, v), do)
    i = torch.arange(T)
    want, _ = mr.attention(q, k, v, see, i[:, None] - i, hd, do=do, dtype=torch.float32)
    for name, r in zip(("o", "dq", "dk", "dv"), (ref.detach(), *g)):
        assert torch.allclose(want[name], r, rtol=1e-10, atol=1e-12), name


def test_the_oracles_ranges():
    assert mr.ranges(1, 6, starts=[0, 2], prefix=[0, 2]) == ([0, 0, 2, 2, 2, 2], [1, 2, 4, 4, 5, 6])
    assert mr.ranges(2, 3, lengths=[2, 5], window=2) == ([0, 0, 0, 3, 3, 4], [1, 2, 0, 4, 5, 6])
    assert mr.ranges(1, 4, starts=[1], lengths=[2], causal=False) == ([0, 1, 1, 0], [0, 3, 3, 0])
