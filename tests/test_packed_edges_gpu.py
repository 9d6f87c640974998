"""The operators of a step over packed documents at the edges of what they take, on the GPU."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_rows_of_no_tokens_have_lengths():
    from femtotron_amd import attention_mask, masked_attention
    zeros = torch.zeros(3, dtype=torch.int64, device=DEV)
    for mask in (attention_mask(3, 0, lengths=zeros), attention_mask(3, 0, lengths=zeros, prefix=zeros), attention_mask(3, 0, zeros, zeros)):
        x = torch.empty(3, 0, 128, dtype=torch.bfloat16, device=DEV)
        assert masked_attention(x, x, x, mask, head_dim=64).shape == x.shape
    with pytest.raises(ValueError, match="3"):
        attention_mask(3, 2, lengths=zeros[:2])
    with pytest.raises(ValueError, match="2"):
        attention_mask(0, 2, zeros[:2], zeros)


def test_clipping_into_outputs_whose_strides_differ_in_dims_of_one():
    """The factor rounds once (2^-24), the product once."""
    from femtotron_amd.optim import clip_gradients
    a = randn((20, 30), 1).to(DEV).t()[None]
    b = torch.empty(600, device=DEV).as_strided((1, 30, 20), (7, 1, 30))
    norm = float(clip_gradients([a], 2.0, out=[b]))
    want = a.double() * (2.0 / (float(a.double().square().sum().sqrt()) + 1e-6))
    assert abs(norm - float(a.double().norm())) <= 2.0 ** -23 * norm
    assert ((b.double() - want).abs() <= 2.0 ** -23 * want.abs()).all()


def test_large_caps_in_fp32_are_none():
    """cap tanh(s / cap) is s to s^3 / (3 cap^2), below fp32's rounding from |s| = 2^-12 cap on."""
    from femtotron_amd import attention_mask, cache_attention, masked_attention
    q, k, v = (randn((1, 70, 128), i).to(DEV) for i in range(3))
    mask, lengths = attention_mask(1, 70, device=DEV), torch.tensor([70], device=DEV)
    plain = masked_attention(q, k, v, mask, head_dim=64)
    one = cache_attention(q[:, -2:], k, v, lengths, head_dim=64)
    # fp32 of scores of up to 2^4 (three roundings of each, 2^-20 all told) and of 128 terms' sums
    bound = 2.0 ** -18 * float(v.abs().max())
    for cap in (1e6, 1e20, 2.0 ** 122):
        assert float((masked_attention(q, k, v, mask, head_dim=64, cap=cap) - plain).abs().max()) <= bound
        assert float((cache_attention(q[:, -2:], k, v, lengths, head_dim=64, cap=cap) - one).abs().max()) <= bound
