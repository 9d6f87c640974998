"""Forward-mode derivatives of block_norms and apply_rotary: refused, not lost.  On the CPU, with the
launches left out (what is tested ends before any output is read)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture
def no_launch(monkeypatch):
    from femtotron_amd import ops
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    monkeypatch.setattr(ops, "_alike", lambda *a: None)
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)


def _block(**dual):
    from femtotron_amd import block_norms
    t = dict(x=torch.randn(4, 64), a=torch.randn(4, 64), w_post=torch.ones(64), w_pre=torch.ones(64), gate=torch.ones(64))
    t.update({k: fwd.make_dual(t[k], torch.ones_like(t[k])) for k in dual})
    return block_norms(t["x"], t["a"], t["w_post"], t["w_pre"], gate=t["gate"])


def _turned(**dual):
    from femtotron_amd import apply_rotary
    t = dict(q=torch.randn(4, 128), k=torch.randn(4, 64))
    t.update({k: fwd.make_dual(t[k], torch.ones_like(t[k])) for k in dual})
    return apply_rotary(t["q"], t["k"], torch.arange(4), torch.ones(32, dtype=torch.float64), head_dim=64)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call,name", [(_block, n) for n in ("x", "a", "w_post", "w_pre", "gate")] + [(_turned, "q"), (_turned, "k")])
def test_a_tangent_is_refused(call, name, grad, no_launch):
    with fwd.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
        call(**{name: True})


def test_without_tangents_the_calls_run(no_launch):
    for call in (_block, _turned):
        assert len(call()) == 2
        with fwd.dual_level():
            assert len(call()) == 2
            with torch.no_grad():
                assert len(call()) == 2


@pytest.mark.gpu
def test_on_the_device():
    from femtotron_amd import apply_rotary, block_norms
    x = torch.randn(4, 64, device="cuda:0")
    w, pos, f = torch.ones(64, device="cuda:0"), torch.arange(4, device="cuda:0"), torch.ones(32, dtype=torch.float64, device="cuda:0")
    h, y = block_norms(x, x, w, w)
    q, _ = apply_rotary(x, None, pos, f, head_dim=64)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            block_norms(d, x, w, w)
        with pytest.raises(NotImplementedError):
            apply_rotary(d, None, pos, f, head_dim=64)
        h2, y2 = block_norms(x, x, w, w)
        q2, _ = apply_rotary(x, None, pos, f, head_dim=64)
    assert torch.equal(h, h2) and torch.equal(y, y2) and torch.equal(q, q2)
