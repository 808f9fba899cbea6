"""Calls of the attention operators that are refused, without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import ternary_vllm_amd as tv


def test_forward_mode_derivatives_are_refused():
    """A dual tensor would come back without its tangent."""
    x, t = torch.zeros(1, 2, 4, 64), torch.zeros(8, 64)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        dt = forward_ad.make_dual(t, torch.ones_like(t))
        ds = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        qkv = forward_ad.make_dual(torch.zeros(1, 2, 256), torch.ones(1, 2, 256))
        for call in (lambda: tv.rotary(d, torch.arange(2), t), lambda: tv.rotary(x, torch.arange(2), dt), lambda: tv.attention(d, x, x), lambda: tv.attention(x, d, x),
                     lambda: tv.attention(x, x, d), lambda: tv.attention(x, x, x, slopes=ds), lambda: tv.cached_attention(d, x, x, 0), lambda: tv.cached_attention(x, d, x, 0),
                     lambda: tv.cached_attention(x, x, d, 0), lambda: tv.rotary_cache(qkv, t, x, x.clone(), 0, 2), lambda: tv.rotary_cache(qkv.detach(), t, d, x, 0, 2)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
