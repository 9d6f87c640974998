"""Activations in 8 bits, without a GPU: the header and its binding, refusals, the oracle's storage."""
from __future__ import annotations

import ctypes
import hashlib
import re

import numpy as np
import pytest
import torch

from oracle import blocks as ob
from tests.conftest import ROOT


def _header() -> str:
    return re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "femtohip_blocks.h").read_text(), flags=re.S)


def _lib():
    from femtotron_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfemtohip.so not built")
    return _lib


def test_library_exports_every_symbol_of_the_blocks_header():
    lib = _lib()
    declared = set(re.findall(r"\b(fh_[a-z0-9_]+)\s*\(", _header()))
    assert declared and declared == set(lib.BLOCK_SIGNATURES), declared ^ set(lib.BLOCK_SIGNATURES)
    raw = ctypes.CDLL(str(lib.LIB_PATH))
    for name in declared:
        assert hasattr(raw, name), name
    assert lib.lib().fh_blocks_abi_version() == lib.BLOCKS_ABI_VERSION


# As ABI_DECLARATIONS of test_api.py: the declarations of a version of this header.
BLOCKS_DECLARATIONS = (1, "1b65722b168f7dcb")


def test_blocks_version_is_raised_with_the_declarations():
    from femtotron_amd import _lib
    text = _header()
    version = int(re.search(r"#define FH_BLOCKS_ABI_VERSION (\d+)", text).group(1))
    text = re.sub(r"#define FH_BLOCKS_ABI_VERSION \d+", "", text)
    digest = hashlib.sha256(re.sub(r"\s+", "", text).encode()).hexdigest()[:16]
    assert (version, digest) == BLOCKS_DECLARATIONS, "declarations changed: raise FH_BLOCKS_ABI_VERSION and record both"
    assert _lib.BLOCKS_ABI_VERSION == version


def test_a_library_without_the_block_operators_is_refused(tmp_path, monkeypatch):
    """One built before them (its own version right) says to rebuild, and is not bound."""
    import subprocess

    lib = _lib()
    src = tmp_path / "old.c"
    src.write_text("int fh_abi_version(void) { return %d; }" % lib.ABI_VERSION)
    so = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    monkeypatch.setattr(lib, "LIB_PATH", so)
    monkeypatch.setattr(lib, "_lib", None)
    with pytest.raises(lib.FemtoHipError, match="rebuild"):
        lib.lib()


def test_packed_calls_are_refused_on_the_host():
    lib = _lib()
    L = lib.lib()
    p = ctypes.c_void_p(1 << 20)  # aligned, never read: every call below is refused before a launch
    off = ctypes.c_void_p((1 << 20) + 4)
    bad = [
        ("fh_pack8", (7, 0, p, p, p, 4, 64, None), b"dtype"),
        ("fh_pack8", (0, 2, p, p, p, 4, 64, None), b"format"),
        ("fh_pack8", (0, 0, p, p, p, 4, 60, None), b"multiple of 8"),
        ("fh_pack8", (0, 0, p, p, p, -1, 64, None), b"rows"),
        ("fh_pack8", (0, 0, p, p, p, 1 << 40, 64, None), b"too many"),
        ("fh_pack8", (0, 0, None, p, p, 4, 64, None), b"null"),
        ("fh_pack8", (0, 0, off, p, p, 4, 64, None), b"aligned"),
        ("fh_unpack8", (0, 0, off, p, p, 4, 64, None), b"aligned"),
        ("fh_unpack8", (0, -1, p, p, p, 4, 64, None), b"format"),
        ("fh_rmsnorm_fwd_pack8", (0, 0, p, p, p, p, p, None, 4, 8200, 1e-5, 0, None), b"8192"),
        ("fh_rmsnorm_fwd_pack8", (0, 0, p, p, p, off, p, None, 4, 64, 1e-5, 0, None), b"aligned"),
        ("fh_rmsnorm_fwd8", (0, 1, p, None, p, p, None, 4, 64, 1e-5, 0, None), b"null"),
        ("fh_rmsnorm_fwd8", (0, 1, p, p, p, p, None, 1 << 26, 64, 1e-5, 0, None), b"2^26"),
        ("fh_add_rmsnorm_fwd8", (0, 1, p, p, p, p, p, p, None, 4, 64, 1e-5, 0, None), b"alias"),
        ("fh_rmsnorm_bwd8", (0, 1, p, p, p, p, None, None, p, p, None, 4, 64, 1e-5, 0, None), b"null"),
        ("fh_rmsnorm_bwd8", (0, 1, p, p, p, p, None, off, p, p, p, 4, 64, 1e-5, 0, None), b"aligned"),
    ]
    for name, args, word in bad:
        assert getattr(L, name)(*args) == 1, name
        assert word in L.fh_last_error(), (name, L.fh_last_error())
    assert L.fh_pack8(0, 0, None, None, None, 0, 64, None) == 0  # empty is a no-op
    assert L.fh_unpack8(1, 1, None, None, None, 0, 64, None) == 0
    assert L.fh_rmsnorm_bwd8_workspace_size(16384, 2048) == L.fh_rmsnorm_bwd_workspace_size(16384, 2048)


def test_front_end_refuses():
    from femtotron_amd import eight_bit_checkpoint, ops
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        ops.pack8(x)
    with pytest.raises(ValueError, match="HIP device"):
        ops.unpack8(ops.Packed8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="int4"):
        eight_bit_checkpoint("int4")
    with pytest.raises(ValueError, match="use_reentrant"):
        eight_bit_checkpoint()(torch.nn.Linear(2, 2), x, use_reentrant=True, debug=True)


def test_off_the_gpu_the_input_is_kept_as_it_is():
    """A call the kernels do not take runs under torch.utils.checkpoint, as with fused_checkpoint."""
    from femtotron_amd import dispatch_counts, eight_bit_checkpoint, reset_dispatch_counts
    from femtotron_amd.training import ActivationCheckpointWrapper
    lin = torch.nn.Linear(8, 8)
    x = torch.randn(3, 8, requires_grad=True)
    reset_dispatch_counts()
    y = ActivationCheckpointWrapper(lin, checkpoint_fn=eight_bit_checkpoint("e4m3"))(x)
    y.sum().backward()
    assert dispatch_counts() == {"fused": 0, "fallback": 1}
    assert torch.equal(y, lin(x)) and torch.allclose(x.grad, lin.weight.sum(0).expand(3, 8))


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """Where the tensors' device is not the current one, the call is made with it current."""
    from contextlib import contextmanager
    from types import SimpleNamespace

    from femtotron_amd import ops
    lib = _lib()
    seen, current = [], [0]

    @contextmanager
    def device(d):
        current[0], old = d, current[0]
        yield
        current[0] = old

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(lib, "lib", lambda: SimpleNamespace(fh_x=lambda *a: seen.append((current[0], a)) or 0))

    class T:
        def __init__(self, i):
            self.get_device = lambda: i

    ops._launch("fh_x", T(0), 1)
    ops._launch("fh_x", T(3), 2)
    assert seen == [(0, (1, 100)), (3, (2, 103))] and current == [0]


@pytest.mark.parametrize("fmt,half", [("int8", 2.0 ** -7), ("e4m3", 2.0 ** -4)])
def test_stored_values_are_near_and_are_held_exactly(fmt, half):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((64, 200)) * np.exp(rng.uniform(-60, 60, (64, 1)))
    x = torch.from_numpy(x).bfloat16().double().numpy()
    codes, exps = ob.pack8(x, fmt)
    back = ob.unpack8(codes, exps)
    pad = np.zeros((64, 224))
    pad[:, :200] = np.abs(x)
    m = np.repeat(pad.reshape(64, 7, 32).max(-1), 32, 1)[:, :200]
    if fmt == "int8":
        assert (np.abs(back - x) <= half * m).all()
        assert np.abs(codes).max() == 127
    else:
        E = np.repeat(exps.astype(int) - 127, 32, 1)[:, :200]
        assert (np.abs(back - x) <= np.maximum(half * np.abs(x), np.ldexp(1.0, E - 10))).all()
        assert np.abs(codes).max() <= 448
    assert (torch.from_numpy(back).bfloat16().double().numpy() == back).all()
