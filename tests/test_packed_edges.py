"""The operators of a step over packed documents at the edges of what they take, without a GPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.test_packed_api import _lib, _mask, no_kernel  # noqa: F401


@pytest.mark.parametrize("cap", [1e-50, 1e-46, 1e39, float("inf"), float("nan"), -1e-50])
def test_a_cap_that_fp32_does_not_hold_is_refused(cap, no_kernel):
    """One that it rounds to 0 would be none."""
    from femtotron_amd import cache_attention, masked_attention
    q, k = torch.randn(4, 128), torch.randn(4, 64)
    for call in (lambda c: masked_attention(q, k, k, _mask(4), head_dim=64, cap=c),
                 lambda c: cache_attention(q[:1, None], k[None], k[None], torch.tensor([3]), head_dim=64, cap=c)):
        call(30.0)
        call(torch.tensor(30.0))
        with pytest.raises(ValueError, match="cap"):
            call(cap)


def test_a_cap_that_is_too_large_for_the_scale_is_refused():
    """cap * log2(e) would overflow, or scale / cap lose its bits."""
    lib = _lib()
    L = lib.lib()

    def status(dt, scale, cap):
        return L.fh_masked_attn_fwd(dt, 16, 64, 16, 64, 16, 64, 16, 64, None, None, 16, 0, 1, 1, 64, scale, cap, None, None)

    for cap in (2.4e38, 2.0 ** 126 * 1.01):
        assert status(1, 1.0, cap) == 1 and b"cap" in L.fh_last_error()
    assert status(1, 1e-3, 1e36) == 1 and b"cap" in L.fh_last_error()
    for dt, scale, cap in ((1, 1.0, 2.0 ** 125), (1, 0.125, 1e6), (1, 2.0 ** -40, 2.0 ** 86), (0, 0.125, 4096.0), (0, 1e-36, 50.0),
                           (1, 0.125, 0.0)):
        assert status(dt, scale, cap) == 0, (dt, scale, cap)


def test_outputs_whose_strides_differ_in_dims_of_one(no_kernel):
    from femtotron_amd.optim import clip_gradients
    a = torch.randn(20, 30).t()[None]                                # strides (600, 1, 30)
    b = torch.empty(20, 30).t().as_strided((1, 30, 20), (7, 1, 30))
    clip_gradients([a, torch.randn(3)], 1.0, out=[b, torch.empty(3)])
    clip_gradients([b], 1.0, out=[a])
    assert no_kernel.count("fh_clip_grads") == 2
    with pytest.raises(ValueError, match="strides"):
        clip_gradients([a], 1.0, out=[torch.empty(1, 30, 20)])


def test_a_norm_that_is_to_be_differentiated_is_refused(no_kernel):
    from femtotron_amd.optim import clip_grad_norm_, gradient_norm
    p = torch.nn.Parameter(torch.ones(5))
    g, = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    with pytest.raises(TypeError, match="derivative"):
        gradient_norm([g.detach(), g])
    with torch.no_grad():
        gradient_norm([g])
    gradient_norm([g.detach()])
    with fwd.dual_level():
        gradient_norm([g.detach()])
        with pytest.raises(TypeError, match="derivative"):
            gradient_norm([fwd.make_dual(g.detach(), torch.ones(5))])
    p.grad = g.detach().clone()
    clip_grad_norm_([p], 1.0)
    assert no_kernel.count("fh_clip_grads") == 4
