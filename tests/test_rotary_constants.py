"""apply_rotary's frequencies and factor are constants: one that wants a gradient is refused instead
of getting none.  On the CPU, with the launches left out."""
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


@pytest.mark.parametrize("leaf", [True, False])
def test_learned_frequencies_and_factors_are_refused(leaf, no_launch):
    from femtotron_amd import apply_rotary, block_norms
    q, pos, f = torch.randn(4, 64, requires_grad=leaf), torch.arange(4), torch.ones(32, dtype=torch.float64)
    learned = f.clone().requires_grad_(True)
    with pytest.raises(TypeError, match="inv_freq"):
        apply_rotary(q, None, pos, learned, head_dim=64)
    with pytest.raises(TypeError, match="factor"):
        apply_rotary(q, None, pos, f, head_dim=64, factor=torch.ones((), requires_grad=True))
    with torch.no_grad():  # no gradient is asked for
        apply_rotary(q, None, pos, learned, head_dim=64)
        apply_rotary(q, None, pos, f, head_dim=64, factor=torch.ones((), requires_grad=True))
    apply_rotary(q, None, pos, learned.detach(), head_dim=64, factor=torch.tensor(1.5))
    with fwd.dual_level():
        with pytest.raises(TypeError, match="inv_freq"):
            apply_rotary(q, None, pos, fwd.make_dual(f, torch.ones_like(f)), head_dim=64)
        one = torch.ones(())
        with pytest.raises(TypeError, match="factor"):
            apply_rotary(q, None, pos, f, head_dim=64, factor=fwd.make_dual(one, one.clone()))
        w = torch.ones(64)
        with pytest.raises(TypeError, match="scale"):
            block_norms(q.detach(), q.detach(), w, scale=fwd.make_dual(one, one.clone()))
