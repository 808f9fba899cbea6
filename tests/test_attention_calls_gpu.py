"""Calls of the attention operators around other parts of torch: forward mode, graph capture."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tv():
    import ternary_vllm_amd
    return ternary_vllm_amd


def test_forward_mode_is_refused_and_a_dual_level_changes_nothing(tv, dev):
    x, table, pos = torch.randn(1, 5, 2, 64, device=dev), tv.rotary_table(32, 5, device=dev), torch.arange(5, device=dev)
    want = tv.attention(tv.rotary(x, pos, table), x, x)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for leaf in (d, forward_ad.make_dual(x.clone().requires_grad_(True), torch.ones_like(x))):
            for call in (lambda: tv.rotary(leaf, pos, table), lambda: tv.attention(leaf, x, x), lambda: tv.attention(x, x, leaf)):
                with pytest.raises(NotImplementedError):
                    call()
        assert torch.equal(tv.attention(tv.rotary(x, pos, table), x, x), want)      # tensors without tangents
    y = x.clone().requires_grad_(True)
    with forward_ad.dual_level():
        (g,) = torch.autograd.grad(tv.attention(y, x, x).sum(), y)
    (h,) = torch.autograd.grad(tv.attention(y, x, x).sum(), y)
    assert torch.equal(g, h)
