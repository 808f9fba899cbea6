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


def test_capture_beside_a_live_graph_of_other_operations_is_refused(tv, dev):
    """The leaf's gradient node was made by another operation of torch, on another stream than the captured one: refused, also if an eager call of
    this module has used the leaf since; once those graphs are gone the capture works."""
    q, k, v = (torch.randn(1, 20, 2, 64, device=dev, requires_grad=True) for _ in range(3))
    table, pos, go = tv.rotary_table(32, 20, device=dev), torch.arange(20, device=dev), torch.randn(1, 20, 2, 64, device=dev)
    odd = torch.randn(1, 20, 2, 128, device=dev)[..., ::2].detach().requires_grad_(True)       # copied inside the call
    s = torch.cuda.Stream()
    for call, leaf in ((lambda: tv.attention(q, k, v), q), (lambda: tv.attention(q, k, v), v), (lambda: tv.rotary(q, pos, table), q), (lambda: tv.rotary(odd, pos, table), odd)):
        alive = leaf * 2
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            more = call()
        torch.cuda.current_stream().wait_stream(s)
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
                call()
        want = more.detach().clone()
        (grad,) = torch.autograd.grad(more, leaf, go)
        del alive, more
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
            (got,) = torch.autograd.grad(out, leaf, go)
        for _ in range(3):
            out.detach().zero_()
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(got, grad)
        del out, got, graph


def test_a_leaf_taken_twice_in_one_capture(tv, dev):
    """Calls of one capture that share leaves, and a second capture on the same stream while the first one's graph is alive."""
    x = torch.randn(1, 20, 4, 64, device=dev, requires_grad=True)
    table, pos, go = tv.rotary_table(32, 20, device=dev), torch.arange(20, device=dev), torch.randn(1, 20, 4, 64, device=dev)

    def step():
        y = tv.attention(tv.rotary(x, pos, table), x, x, causal=True) + tv.attention(x, x, x)
        return [y, *torch.autograd.grad(y, x, go)]

    want = [y.detach().clone() for y in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            outs.append(step())
    for n in range(4):
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs[n % 2])), n


def test_rotary_cache_refuses_interleaved_caches_that_share_slots(tv, dev):
    table, qkv = tv.rotary_table(16, 9, device=dev), torch.randn(2, 3, 8 * 16, device=dev)
    both = torch.zeros(2, 5, 9, 16, device=dev)
    for k, v in ((both[:, :2], both[:, 1:3]), (both[:, 2:4], both[:, 1:3])):
        with pytest.raises(ValueError, match="share"):
            tv.rotary_cache(qkv, table, k, v, 0, 4)
    k, v = torch.zeros(2, 2, 9, 16, device=dev), torch.zeros(2, 2, 9, 16, device=dev)
    want = tv.rotary_cache(qkv, table, k, v, 4, 4)
    assert torch.equal(tv.rotary_cache(qkv, table, both[:, :2], both[:, 2:4], 4, 4), want)
    assert torch.equal(both[:, :2], k) and torch.equal(both[:, 2:4], v) and int(both[:, 4].count_nonzero()) == 0
