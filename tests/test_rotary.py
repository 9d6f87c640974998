"""Rotary positions without a GPU: frequencies against Hugging Face's, refusals."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("dim,theta", [(64, 1e4), (128, 5e5), (16, 1e4)])
@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0}, LLAMA3, {"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "mscale": 0.707, "mscale_all_dim": 1.0, "beta_fast": 16},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, "truncate": False, "attention_factor": 1.5},
    {"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 2048}])
def test_frequencies_are_hugging_faces(dim, theta, scaling):
    """HF computes them in fp32: a power (exponents to 13.2, so 2^-24 * 13.2 relative), and a
    ramp with a few roundings of values up to 40."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    from femtotron_amd import rotary_frequencies
    cfg = LlamaConfig(hidden_size=dim * 4, num_attention_heads=4, max_position_embeddings=2048, rope_theta=theta,
                      rope_scaling=dict(scaling))
    kind = scaling.get("rope_type", scaling.get("type"))
    ref, factor = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=8192)
    got, f = rotary_frequencies(dim, theta, scaling, seq_len=8192)
    assert got.dtype == torch.float64 and got.shape == (dim // 2,)
    assert math.isclose(f, factor, rel_tol=1e-12)
    assert float((got / ref.double() - 1).abs().max()) <= 2.0 ** -24 * (13.2 + 40)


def test_frequencies_unscaled_and_refused():
    from femtotron_amd import rotary_frequencies
    f, factor = rotary_frequencies(8, 16.0)
    assert factor == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.5, 0.25, 0.125], dtype=torch.float64), rtol=1e-15)
    # a sequence within the original context is not stretched
    d = {"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 2048}
    assert torch.equal(rotary_frequencies(64, 1e4, d, seq_len=100)[0], rotary_frequencies(64, 1e4)[0])
    for bad, word in ((dict(rot_dim=7), "even"), (dict(rot_dim=0), "even"), (dict(rot_dim=8, theta=0.5), "theta"),
                      (dict(rot_dim=8, scaling={"rope_type": "longrope"}), "rope_type"),
                      (dict(rot_dim=8, scaling={"rope_type": "linear"}), "factor"),
                      (dict(rot_dim=8, scaling={**LLAMA3, "high_freq_factor": 1.0}), "high_freq_factor")):
        with pytest.raises(ValueError, match=word):
            rotary_frequencies(**bad)


def test_calls_are_refused_on_the_host():
    from femtotron_amd import _lib, ops
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfemtohip.so not built")
    L = _lib.lib()
    p, r = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 24)  # never read: every call below is refused before a launch
    ok = dict(dt=0, q=p, ldq=256, nq=4, k=r, ldk=128, nk=2, qo=p, ldqo=256, ko=r, ldko=128, tokens=6, hd=64, rot=64,
              off=0, layout=0, pos=p, npos=6, f=p, factor=1.0, stream=None)
    for change, word in ((dict(dt=5), b"dtype"), (dict(layout=2), b"layout"), (dict(tokens=-1), b"tokens"),
                         (dict(nq=-1), b"heads"), (dict(hd=0), b"head_dim"), (dict(hd=2048, rot=64), b"head_dim"),
                         (dict(rot=63), b"rot_dim"), (dict(rot=0), b"rot_dim"), (dict(off=2), b"rot_dim"),
                         (dict(ldq=255), b"stride"), (dict(ldko=64), b"stride"), (dict(k=None), b"null"),
                         (dict(pos=None), b"null"), (dict(f=None), b"null"), (dict(npos=4), b"n_positions"),
                         (dict(npos=0), b"n_positions"), (dict(ldqo=512), b"in place"), (dict(nq=1 << 20, ldq=1 << 30, ldqo=1 << 30), b"2^20"),
                         (dict(ldq=1 << 29, ldqo=1 << 29), b"2^28"),
                         (dict(q=ctypes.c_void_p((1 << 22) + 1)), b"aligned"), (dict(qo=r), b"overlap"),
                         (dict(ko=ctypes.c_void_p((1 << 20) + 2 * 255)), b"overlap"),
                         (dict(qo=ctypes.c_void_p((1 << 20) + 2)), b"overlap"), (dict(nq=1 << 30), b"heads"),
                         (dict(pos=ctypes.c_void_p((1 << 20) + 4)), b"aligned"), (dict(off=1 << 62), b"rot_dim"),
                         (dict(tokens=1 << 40, npos=1 << 20), b"too many")):
        for name in ("fh_rotary_fwd", "fh_rotary_bwd"):
            assert getattr(L, name)(*{**ok, **change}.values()) == 1, change
            assert word in L.fh_last_error(), (change, L.fh_last_error())
    assert L.fh_rotary_fwd(*{**ok, "tokens": 0, "q": None}.values()) == 0
    with pytest.raises(ValueError, match="HIP device"):
        ops.rotary_fwd(torch.zeros(2, 64), None, torch.arange(2), torch.ones(32, dtype=torch.float64), head_dim=64)


def test_block_norms_are_refused_on_the_host():
    from femtotron_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfemtohip.so not built")
    L = _lib.lib()
    p, q, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 21), ctypes.c_void_p((1 << 20) + 8)
    fwd = dict(dt=0, x=p, a=p, w1=p, w2=p, g=None, per=0, s=1.0, h=q, y=q, r1=None, r2=None, rows=4, cols=64, eps=1e-5,
               stream=None)
    for change, word in ((dict(dt=2), b"dtype"), (dict(cols=60), b"multiple of 8"), (dict(cols=8200), b"8192"),
                         (dict(rows=-1), b"rows"), (dict(w1=None, w2=None), b"at least one"), (dict(a=None), b"null"),
                         (dict(y=None), b"null"), (dict(x=odd), b"aligned"), (dict(h=p), b"alias")):
        assert L.fh_block_norms_fwd(*{**fwd, **change}.values()) == 1, change
        assert word in L.fh_last_error(), (change, L.fh_last_error())
    assert L.fh_block_norms_fwd(*{**fwd, "rows": 0, "x": None}.values()) == 0
    r = ctypes.cast(p, ctypes.POINTER(ctypes.c_float))
    bwd = dict(dt=0, dh=p, dy=p, h=p, a=p, w1=p, w2=p, g=p, per=0, s=1.0, r1=r, r2=r, dx=q, da=q, dw1=q, dw2=q, dg=q,
               ws=q, rows=4, cols=64, stream=None)
    for change, word in ((dict(dh=None), b"null"), (dict(dy=None), b"dy"), (dict(r1=None), b"rstd_post"), (dict(r2=None), b"rstd_pre"),
                         (dict(a=None), b"a with"), (dict(dg=None), b"null"), (dict(dg=None, per=1), b"dgate"),
                         (dict(ws=None), b"null"), (dict(ws=odd), b"aligned"), (dict(dw2=None), b"null")):
        assert L.fh_block_norms_bwd(*{**bwd, **change}.values()) == 1, change
        assert word in L.fh_last_error(), (change, L.fh_last_error())
    assert L.fh_block_norms_bwd_workspace_size(0, 64) == 0
    assert L.fh_block_norms_bwd_workspace_size(16384, 2048) > 0
