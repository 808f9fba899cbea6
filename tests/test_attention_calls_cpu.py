"""Calls of the attention operators that are refused, without a GPU."""
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import ternary_vllm_amd as tv  # noqa: E402
from test_attention_cpu import P, attention_args, grads_args  # noqa: E402


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


def test_which_leaves_another_graph_holds():
    """What a recorded call asks about its leaves: a node that lives because some graph holds it, whichever operation made it, unless marked as of the same stream."""
    held = tv.attention_ops._held
    x = torch.zeros(3, requires_grad=True)
    assert not held(x, 7) and not held(x, 7)             # asking leaves nothing behind
    y = x * 2
    assert held(x, 7) and held(x, 7)
    torch.autograd.graph.get_gradient_edge(x).node.metadata["tvl_stream"] = 7
    assert not held(x, 7) and held(x, 8)
    del y
    assert not held(x, 8)
    (x * 2).sum().backward()
    assert not held(x, 7)


@pytest.mark.parametrize("batch,heads,tokens", [(1 << 20, 12, 1), (1 << 19, 16, 1), (1 << 20, 8, 64), (1 << 15, 16, 2048), (1, 8, 1 << 27)])
def test_gradient_launches_beyond_the_grid_are_refused(batch, heads, tokens):
    """The gradient kernels start up to 512 threads for every 128 rows: 2^32 threads are refused before anything is launched, by the forward call that
    precedes them too."""
    lib = tv.custom_ops_mod._lib
    for dim in (64, 128):
        a = attention_args(batch=batch, heads=heads, kv_heads=heads, queries=tokens, keys=tokens, dim=dim, o_batch=tokens * heads * dim, o_token=heads * dim, o_head=dim)
        assert lib.tvl_attention_backward(a, grads_args(), P, 1 << 62, None) == 1 and b"too many" in lib.tvl_last_error()
        assert lib.tvl_attention(a, None, 0, None) == 1 and b"too many" in lib.tvl_last_error()


def test_views_that_share_elements_are_found():
    """Against the sets of their elements, for layouts of caches: heads beside each other, slots apart, layers of one tensor."""
    meet, apart = tv.attention_ops._meet, tv.attention_ops._apart
    big = torch.zeros(6, 4, 5, 7, 8)
    views = [big[i:i + 2, h:h + 2, b, s:s + 4:st, e:e + 3] for i in (0, 1, 2) for h in (0, 1, 2) for b in (0, 1) for s, st in ((0, 1), (3, 1), (0, 2), (1, 2)) for e in (0, 2, 5)]
    places = [set((torch.arange(big.numel()).view(big.shape).as_strided(v.shape, v.stride(), v.storage_offset())).flatten().tolist()) for v in views]
    found = 0
    for x, px in zip(views[::3], places[::3]):
        assert apart(x)
        for y, py in zip(views, places):
            if x.stride() == y.stride() and x.shape == y.shape:
                assert meet(x, y) == bool(px & py), (x.storage_offset(), y.storage_offset(), x.stride())
                found += bool(px & py)
    assert found > 100
    assert not meet(views[0], views[0].clone()) and not meet(big[:, 0], big.clone()[:, 0])


@pytest.mark.parametrize("scale,softcap", [(1e39, 0.0), (-1e39, 0.0), (float("inf"), 0.0), (float("nan"), 0.0), (1.0, 1e39), (1.0, float("inf")), (1.0, float("nan")), (1.0, -1.0)])
def test_scales_and_caps_beyond_float32_are_refused(scale, softcap):
    with pytest.raises(ValueError, match="scale"):
        tv.attention_ops._scale_cap(scale, softcap, 64, "attention")
    assert tv.attention_ops._scale_cap(3e38, 3e38, 64, "attention") == (3e38, 3e38)
