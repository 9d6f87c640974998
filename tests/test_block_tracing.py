"""The operators around a block under torch.jit.trace and make_fx, which see no kernel: refused, or the
trace would return uninitialised memory."""
from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture
def no_kernel(monkeypatch):
    """Everything up to the entry point, which counts its calls; tensors on the CPU."""
    from femtotron_amd import _lib, ops
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: 64 if name.endswith("_workspace_size") else calls.append(name) or 0

    monkeypatch.setattr(ops, "_alike", lambda *a: None)
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    return calls


def _calls():
    from femtotron_amd import apply_rotary, block_norms, ops
    x, w, f = torch.randn(4, 64), torch.ones(64), torch.ones(32, dtype=torch.float64)
    pos, r = torch.arange(4), torch.ones(4)
    p = ops.Packed8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8))
    return {
        "block_norms": lambda t: block_norms(t, t, w, w)[0],
        "block_norms_fwd": lambda t: ops.block_norms_fwd(t, t, w, w, 1e-5)[0],
        "block_norms_bwd": lambda t: ops.block_norms_bwd(t, t, t, t, w, w, rstd_post=r, rstd_pre=r)[0],
        "apply_rotary": lambda t: apply_rotary(t, None, pos, f, head_dim=64)[0],
        "rotary_bwd": lambda t: ops.rotary_bwd(t, None, pos, f, head_dim=64)[0],
        "pack8": lambda t: ops.pack8(t).codes,
        "rmsnorm_fwd_pack8": lambda t: ops.rmsnorm_fwd_pack8(t, w, 1e-5)[0],
        "add_rmsnorm_fwd8": lambda t: ops.add_rmsnorm_fwd8(p, t, w, 1e-5)[0],
        "rmsnorm_bwd8": lambda t: ops.rmsnorm_bwd8(t, p, w, 1e-5)[0],
    }, x


NAMES = ("block_norms", "block_norms_fwd", "block_norms_bwd", "apply_rotary", "rotary_bwd", "pack8", "rmsnorm_fwd_pack8",
         "add_rmsnorm_fwd8", "rmsnorm_bwd8")


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
def test_a_trace_is_refused(name, no_kernel, monkeypatch):
    from femtotron_amd import ops
    monkeypatch.setattr(ops, "_packed", lambda name, p: (0, 4, 64))
    monkeypatch.setattr(ops, "_norm8_args", lambda *a: 0)
    calls, x = _calls()
    with pytest.raises(RuntimeError, match="torch.jit"):
        torch.jit.trace(calls[name], (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(calls[name])(x)
    assert no_kernel == []
    calls[name](x)  # untraced it reaches its entry point
    assert len(no_kernel) == 1


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", ["block_norms", "apply_rotary"])
def test_a_trace_that_wants_gradients_is_refused(name, no_kernel):
    calls, x = _calls()
    with pytest.raises(RuntimeError, match="torch.jit"):
        torch.jit.trace(calls[name], (x.requires_grad_(True),), check_trace=False)
    assert no_kernel == []
