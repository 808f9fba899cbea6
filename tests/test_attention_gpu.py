"""The attention operators on the GPU against their float64 definition (tests/attention_reference.py), within bounds built from the
roundings the kernels make."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attention_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tv():
    import ternary_vllm_amd
    return ternary_vllm_amd


def normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------------------- rotary

def rotate64(x, table, interleaved, inverse=False):
    """x [..., d] float64, table rows [..., rd] of the same leading shape."""
    half = table.shape[-1] // 2
    cos, sin = table[..., :half].double(), table[..., half:].double() * (-1 if inverse else 1)
    part = x[..., : 2 * half].double()
    a, c = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    u, w = a * cos - c * sin, c * cos + a * sin
    part = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    size = torch.cat([part.abs() * 0 + (a.abs() + c.abs()).repeat_interleave(2, -1) if interleaved else torch.cat([a.abs() + c.abs()] * 2, -1), x[..., 2 * half:].abs().double()], -1)
    return torch.cat([part, x[..., 2 * half:].double()], -1), size


def check_rotary(got, x, table, interleaved, inverse=False, what=""):
    want, size = rotate64(x, table, interleaved, inverse)
    u = R.unit(x.dtype)
    # float32 products and sum (three roundings of at most |a| + |c| times the amplitude), then one rounding; float16 subnormals round by 2^-25
    R.within(got, want, 3 * R.F32 * size * 1.5 + u * want.abs() * 1.01 + (2.0 ** -25 if x.dtype == torch.float16 else 0), what)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,h,d,rd", [(1, 1, 1, 64, 32), (2, 7, 3, 64, 64), (2, 33, 5, 80, 32), (3, 5, 2, 33, 10), (1, 130, 4, 128, 48), (2, 4, 3, 20, 0), (1, 3, 2, 6, 6)])
def test_rotary_forward_and_gradient(tv, dev, kind, interleaved, b, t, h, d, rd):
    g = torch.Generator().manual_seed(b * 1000 + d + rd)
    x, gy = normal(g, b, t, h, d, dtype=TYPES[kind]), normal(g, b, t, h, d, dtype=TYPES[kind])
    table = tv.rotary_table(rd, 300, device=dev)
    shared = torch.randperm(300, generator=g)[:t] if rd else torch.arange(t)
    own = torch.randint(0, 300, (b, t), generator=g)            # the same position may come twice
    for pos in (shared, own):
        rows = table.cpu()[pos if pos.dim() == 2 else pos[None].expand(b, t)][:, :, None].expand(b, t, h, rd)
        leaf = x.to(dev).requires_grad_(True)
        y = tv.rotary(leaf, pos.to(dev), table, interleaved=interleaved)
        check_rotary(y, x, rows, interleaved, what="forward")
        (gx,) = torch.autograd.grad(y, leaf, gy.to(dev))
        check_rotary(gx, gy, rows, interleaved, inverse=True, what="gradient")
        with torch.no_grad():
            assert torch.equal(tv.rotary(leaf, pos.to(dev), table, interleaved=interleaved), y)


def test_rotary_strides_alignment_and_gradient_layouts(tv, dev):
    g = torch.Generator().manual_seed(3)
    table = tv.rotary_table(32, 64, device=dev)
    wide = torch.cat([table, table], 1)[:, :32]                    # rows further apart than they are long
    big = normal(g, 2, 9, 3 * 4 * 64 + 5, dtype=torch.float16).to(dev)
    pos = torch.arange(9, device=dev)
    views = [big[..., :256].view(2, 9, 4, 64) if False else big[..., :256].unflatten(-1, (4, 64)),        # heads inside a longer row, odd row length
             big[..., 1:257].unflatten(-1, (4, 64)),                                                            # off a 16-byte boundary
             big[..., :512].unflatten(-1, (8, 64))[:, :, ::2],                                                 # every second head
             big[..., :256].unflatten(-1, (4, 64)).transpose(0, 1).contiguous().transpose(0, 1),                # tokens outside batch
             big[..., :512].unflatten(-1, (4, 128))[..., ::2]]                                                  # not dense in the head: copied
    for x in views:
        want = tv.rotary(x.contiguous(), pos, table)
        assert torch.equal(tv.rotary(x, pos, table), want) and torch.equal(tv.rotary(x, pos, wide), want)
    x = views[0].detach().requires_grad_(True)
    y = tv.rotary(x, pos, table)
    (a,) = torch.autograd.grad(y.sum(), x)                         # an expanded gradient
    (b,) = torch.autograd.grad(tv.rotary(x, pos, table), x, torch.ones_like(y))
    assert torch.equal(a, b)
    every = torch.arange(18, device=dev).view(2, 9)
    assert torch.equal(tv.rotary(views[0], every.t().contiguous().t(), table), tv.rotary(views[0], every, table))


def test_rotary_positions_outside_the_table_give_nan_and_refusals(tv, dev):
    table = tv.rotary_table(32, 10, device=dev)
    x = torch.randn(2, 4, 3, 64, device=dev)
    pos = torch.tensor([[0, -1, 9, 10], [1 << 40, 3, -(1 << 40), 2]], device=dev)
    y = tv.rotary(x, pos, table)
    bad = (pos < 0) | (pos >= 10)
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert tv.rotary(x[:, :0], pos[:, :0], table).shape == (2, 0, 3, 64)
    for call in (lambda: tv.rotary(x, pos.int(), table), lambda: tv.rotary(x, pos[:, :3], table), lambda: tv.rotary(x, pos, table.half()), lambda: tv.rotary(x[0], pos, table),
                 lambda: tv.rotary(x, pos, tv.rotary_table(66, 10, device=dev)), lambda: tv.rotary(x, pos, table.clone().requires_grad_(True)), lambda: tv.rotary(x.double(), pos, table),
                 lambda: tv.rotary(x, pos.cpu(), table)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,hq,hk,d,rd", [(1, 1, 4, 4, 64, 32), (3, 9, 4, 2, 64, 64), (2, 5, 3, 1, 33, 10), (2, 17, 8, 1, 128, 128)])
def test_rotary_cache_writes_only_its_slots(tv, dev, kind, interleaved, b, t, hq, hk, d, rd):
    g = torch.Generator().manual_seed(17 + d)
    slots, dt = 40, TYPES[kind]
    row = (hq + 2 * hk) * d
    qkv = normal(g, b, t, row + 3, dtype=dt)                        # a longer row, as of a product with more channels
    kc, vc = normal(g, b, hk, slots, d, dtype=dt), normal(g, b, hk, slots, d, dtype=dt)
    table = tv.rotary_table(rd, slots, device=dev)
    before = torch.randint(0, slots - t + 1, (b,), generator=g)
    count = torch.randint(0, t + 1, (b,), generator=g)
    count[0] = t
    for lens, n in ((before, None), (before, count), (torch.tensor(7), None), (5, count)):
        k, v = kc.to(dev), vc.to(dev)
        at = lens if isinstance(lens, int) else lens.to(dev)
        q = tv.rotary_cache(qkv.to(dev)[..., :row + 3], table, k, v, at, hq, interleaved=interleaved, count=None if n is None else n.to(dev))
        assert q.shape == (b, t, hq, d)
        starts = [lens] * b if isinstance(lens, int) else (lens.tolist() if lens.dim() else [int(lens)] * b)
        reals = [t] * b if n is None else n.tolist()
        wk, wv = kc.clone(), vc.clone()
        for i in range(b):
            s, c = starts[i], reals[i]
            x = qkv[i, :, :row].unflatten(-1, (hq + 2 * hk, d))
            rows = table.cpu()[s: s + c][:, None].expand(c, hq + hk, rd)
            both = torch.cat([q[i, :c].cpu(), k[i, :, s: s + c].transpose(0, 1).cpu()], 1)
            if c:
                check_rotary(both, x[:c, : hq + hk], rows, interleaved, what="q and k")
            assert int(q[i, c:].count_nonzero()) == 0
            wk[i, :, s: s + c] = k[i, :, s: s + c].cpu()
            wv[i, :, s: s + c] = x[:c, hq + hk:].transpose(0, 1)
        assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)      # every other slot as it was


def test_rotary_cache_positions_outside_and_refusals(tv, dev):
    table = tv.rotary_table(16, 12, device=dev)
    qkv = torch.randn(5, 3, 4 * 32, device=dev)
    k, v = (torch.randn(5, 1, 10, 32, device=dev) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    lens = torch.tensor([-1, 8, 10, 1 << 62, -(1 << 62)], device=dev)
    q = tv.rotary_cache(qkv, table, k, v, lens, 2)
    place = lens[:, None] + torch.arange(3, device=dev)
    bad = (lens[:, None] < 0) | (place >= 10)
    assert torch.isnan(q[bad]).all() and torch.isfinite(q[~bad]).all()
    assert torch.equal(k[[0, 2, 3, 4]], k0[[0, 2, 3, 4]]) and torch.equal(k[1, :, :8], k0[1, :, :8]) and not torch.equal(k[1, :, 8:], k0[1, :, 8:])
    assert torch.equal(v[1, 0, 8:], qkv[1, :2, 96:])
    short = tv.rotary_table(16, 9, device=dev)                       # a table shorter than the cache
    assert torch.isnan(tv.rotary_cache(qkv, short, k0.clone(), v0.clone(), 7, 2)[:, 2]).all()
    cases = [lambda: tv.rotary_cache(qkv, table, k, v, 8, 2), lambda: tv.rotary_cache(qkv, table, k, v, -1, 2), lambda: tv.rotary_cache(qkv, table, k, v, lens.int(), 2),
             lambda: tv.rotary_cache(qkv, table, k, v, lens[:4], 2), lambda: tv.rotary_cache(qkv, table, k, v, 0, 3), lambda: tv.rotary_cache(qkv, table, k, k, 0, 2),
             lambda: tv.rotary_cache(qkv, table, k.half(), v, 0, 2), lambda: tv.rotary_cache(qkv, table, k[:1].expand(5, 1, 10, 32), v, 0, 2),
             lambda: tv.rotary_cache(qkv, table, k[..., :16], v[..., :16], 0, 2, count=lens.float()), lambda: tv.rotary_cache(qkv, table, k, v[:, :, :9], 0, 2),
             lambda: tv.rotary_cache(qkv.clone().requires_grad_(True), table, k, v, 0, 2), lambda: tv.rotary_cache(qkv[0], table, k, v, 0, 2)]
    for call in cases:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rotary_cache_without_query_heads(tv, dev, kind):
    """Keys and values alone: the caches get what they get beside query heads."""
    g = torch.Generator().manual_seed(5)
    qkv = normal(g, 2, 3, 8 * 16, dtype=TYPES[kind]).to(dev)
    table = tv.rotary_table(16, 9, device=dev)
    k, v, k1, v1 = (torch.zeros(2, 2, 9, 16, dtype=TYPES[kind], device=dev) for _ in range(4))
    tv.rotary_cache(qkv, table, k, v, 4, 4)
    q = tv.rotary_cache(qkv[..., 4 * 16:], table, k1, v1, 4, 0)
    assert q.shape == (2, 3, 0, 16) and torch.equal(k, k1) and torch.equal(v, v1) and torch.equal(v1[:, :, 4:7], qkv[..., 6 * 16:].unflatten(2, (2, 16)).transpose(1, 2))


def test_rotary_cache_refuses_caches_that_share_memory(tv, dev):
    table, qkv, kv = tv.rotary_table(16, 9, device=dev), torch.zeros(2, 3, 8 * 16, device=dev), torch.zeros(3, 2, 9, 16, device=dev)
    for k, v in ((kv[:2], kv[:2]), (kv[:2], kv[1:]), (kv[1:], kv[:2])):
        with pytest.raises(ValueError, match="share"):
            tv.rotary_cache(qkv, table, k, v, 0, 4)
    both = torch.zeros(2, 2, 2, 9, 16, device=dev)      # side by side in one tensor: fine
    tv.rotary_cache(qkv, table, both[:, 0], both[:, 1], 0, 4)


# ---------------------------------------------------------------------------------------------------------- attention

def run_case(tv, dev, kind, b, tq, tk, hq, hk, d, causal=False, prefix=None, documents=None, softcap=0.0, slopes=False, scale=None, seed=0, gscale=0.02, qscale=1.0):
    g = torch.Generator().manual_seed(seed + 7 * tq + 13 * tk + d)
    dt = TYPES[kind]
    q, k, v, go = normal(g, b, tq, hq, d, dtype=dt, scale=qscale), normal(g, b, tk, hk, d, dtype=dt), normal(g, b, tk, hk, d, dtype=dt), normal(g, b, tq, hq, d, dtype=dt, scale=gscale)
    sl = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)]) if slopes else None
    pre = torch.zeros(b, dtype=torch.int64) if prefix is None else (torch.full((b,), prefix) if isinstance(prefix, int) else prefix)
    see, place = R.sees(b, tq, tk, causal, pre, documents)
    ref = R.Attention(q, k, v, see, place, scale, softcap, sl)
    leaves = [x.to(dev).requires_grad_(True) for x in (q, k, v)]
    on = lambda x: x.to(dev) if isinstance(x, torch.Tensor) else x
    kw = dict(causal=causal, scale=scale, softcap=softcap, slopes=on(sl), prefix=on(prefix), documents=on(documents))
    out = tv.attention(*leaves, **kw)
    R.within(out, *ref.forward(), what="out")
    grads = torch.autograd.grad(out, leaves, go.to(dev))
    for name, got, (want, tol) in zip(("dq", "dk", "dv"), grads, ref.grads(go)):
        R.within(got, want, tol, name)
    with torch.no_grad():
        assert torch.equal(tv.attention(*leaves, **kw), out)
    again = torch.autograd.grad(tv.attention(*leaves, **kw), leaves, go.to(dev))
    assert all(torch.equal(x, y) for x, y in zip(grads, again))       # the same bits on every call
    return ref, out, grads


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("b,tq,tk,hq,hk,d,causal", [
    (1, 1, 1, 1, 1, 64, True), (2, 1, 1, 4, 2, 8, False), (1, 1, 70, 2, 1, 64, False), (2, 33, 33, 4, 4, 64, True), (1, 64, 64, 2, 2, 32, False), (2, 65, 65, 3, 1, 64, True),
    (1, 130, 130, 4, 2, 128, True), (2, 197, 197, 3, 3, 64, False), (1, 257, 257, 2, 1, 96, True), (1, 100, 300, 2, 2, 64, True), (1, 300, 100, 2, 2, 64, True),
    (1, 129, 31, 2, 1, 80, False), (1, 40, 40, 2, 2, 1, True), (2, 50, 50, 2, 1, 33, True), (1, 70, 70, 2, 2, 127, False), (1, 513, 513, 1, 1, 64, True)])
def test_attention_shapes(tv, dev, kind, b, tq, tk, hq, hk, d, causal):
    ref, out, _ = run_case(tv, dev, kind, b, tq, tk, hq, hk, d, causal)
    if tq > tk and causal:
        assert int(out[:, : tq - tk].count_nonzero()) == 0                # queries in front of the first key see nothing


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("softcap,slopes,prefix,scale", [(30.0, False, None, None), (2.0, True, None, 1.0), (0.0, True, None, None), (0.0, False, 50, None), (5.0, True, 129, 0.3),
                                                           (0.0, False, 1000, None), (0.0, False, None, -0.125), (0.0, False, None, 0.0)])
def test_attention_scores(tv, dev, kind, softcap, slopes, prefix, scale):
    for t, d in ((150, 64), (90, 128)):
        run_case(tv, dev, kind, 2, t, t, 4, 2, d, True, prefix, None, softcap, slopes, scale, seed=1)
    if prefix is None:
        run_case(tv, dev, kind, 1, 70, 140, 2, 2, 64, False, None, None, softcap, slopes, scale, seed=2)


@pytest.mark.parametrize("kind", TYPES)
def test_attention_prefix_per_sequence(tv, dev, kind):
    run_case(tv, dev, kind, 4, 140, 140, 2, 1, 64, True, torch.tensor([0, 1, 77, 200]), seed=3)
    run_case(tv, dev, kind, 2, 90, 140, 2, 1, 64, True, torch.tensor([100, -5]), seed=3)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_documents(tv, dev, kind, causal):
    t = 330
    ids = torch.arange(t)
    packed = torch.where(ids < 100, 0, torch.where(ids < 101, 5, torch.where(ids < 256, 7, 9)))
    packed[310:] = -1
    mixed = ids % 3 - 1                                                # interleaved documents, one of them padding
    ref, out, grads = run_case(tv, dev, kind, 2, t, t, 4, 2, 64, causal, None, torch.stack([packed, mixed]), seed=4)
    assert int(out[0, 310:].count_nonzero()) == 0 and int(out[1, ::3].count_nonzero()) == 0
    assert all(int(x[0, 310:].count_nonzero()) == 0 and int(x[1, ::3].count_nonzero()) == 0 for x in grads)
    run_case(tv, dev, kind, 1, t, t, 2, 1, 128, causal, 120 if causal else None, packed[None], 20.0, True, seed=5)
    run_case(tv, dev, kind, 1, 64, 64, 2, 1, 64, causal, None, torch.full((1, 64), -1), seed=5)          # nobody sees anybody


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("gscale", [1e-4, 300.0])
def test_attention_gradients_of_small_and_large_losses(tv, dev, kind, gscale):
    run_case(tv, dev, kind, 1, 400, 400, 2, 1, 64, True, seed=6, gscale=gscale)


@pytest.mark.parametrize("kind", TYPES)
def test_attention_far_scores(tv, dev, kind):
    """Large scores: one weight takes everything, the maximum moves from tile to tile."""
    run_case(tv, dev, kind, 1, 200, 200, 2, 2, 64, True, seed=7, qscale=12.0)


def test_attention_gradient_against_differences(tv, dev):
    """Along random directions, central differences of the float64 definition against the kernels' float32 gradients."""
    g = torch.Generator().manual_seed(11)
    b, t, hq, hk, d, cap = 1, 37, 4, 2, 24, 3.0
    q, k, v, go = (normal(g, b, t, h, d) for h in (hq, hk, hk, hq))
    sl = torch.tensor([0.5, 0.1, 0.02, 0.0])
    see, place = R.sees(b, t, t, True, torch.tensor([9]), None)
    f = lambda q, k, v: float((R.Attention(q, k, v, see, place, None, cap, sl).out.transpose(1, 2) * go.double()).sum())
    leaves = [x.to(dev).requires_grad_(True) for x in (q, k, v)]
    out = tv.attention(*leaves, causal=True, softcap=cap, slopes=sl.to(dev), prefix=9)
    grads = torch.autograd.grad(out, leaves, go.to(dev))
    for n, x in enumerate((q, k, v)):
        for _ in range(3):
            u = torch.randn(x.shape, generator=g, dtype=torch.float64)
            h = 1e-5
            at = lambda s: f(*[y.double() + s * u if m == n else y.double() for m, y in enumerate((q, k, v))])
            want = (at(h) - at(-h)) / (2 * h)
            got = float((grads[n].cpu().double() * u).sum())
            size = float((grads[n].cpu().double() * u).abs().sum())
            # float32 gradients (relative 1e-5 of the sum's terms) and the difference's own h^2 term
            assert abs(got - want) <= 1e-5 * size + 1e-7, (n, got, want)


@pytest.mark.parametrize("kind", TYPES)
def test_attention_strides_and_alignment(tv, dev, kind):
    """Operands as views: a joint projection, heads outside tokens, rows off 16-byte boundaries, shared and expanded rows, gradients of any layout."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(21)
    b, t, h, d = 2, 75, 2, 64
    qkv = normal(g, b, t, 3 * h * d + 3, dtype=dt).to(dev)
    go = normal(g, b, h, t, d, dtype=dt).to(dev).transpose(1, 2)
    cut = lambda x, o: x[..., o: o + h * d].unflatten(-1, (h, d))
    layouts = [[cut(qkv, o) for o in (0, h * d, 2 * h * d)], [cut(qkv, o + 1) for o in (0, h * d, 2 * h * d)],
               [cut(qkv, o).transpose(1, 2).contiguous().transpose(1, 2) for o in (0, h * d, 2 * h * d)],
               [cut(qkv, 0), cut(qkv, h * d)[:, :, :1].expand(b, t, h, d), cut(qkv, h * d)[:1].expand(b, t, h, d)],
               [torch.stack([cut(qkv, o)] * 2, -1)[..., 0] for o in (0, h * d, 2 * h * d)]]
    for ops3 in layouts:
        for grad in (go, go.contiguous(), go[..., :1].expand(b, t, h, d)):
            views = [x.detach().requires_grad_(True) for x in ops3]
            dense = [x.detach().contiguous().requires_grad_(True) for x in ops3]
            a, c = tv.attention(*views, causal=True), tv.attention(*dense, causal=True)
            assert torch.equal(a, c)
            for x, y in zip(torch.autograd.grad(a, views, grad), torch.autograd.grad(c, dense, grad.contiguous())):
                assert torch.equal(x, y)


def test_attention_partial_gradients_and_leaf_in_place(tv, dev):
    g = torch.Generator().manual_seed(22)
    q, k, v = (normal(g, 1, 70, h, 64).to(dev) for h in (4, 2, 2))
    full = [x.clone().requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(tv.attention(*full, causal=True).square().sum(), full)
    for n in range(3):
        some = [x.clone().requires_grad_(m == n) for m, x in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(tv.attention(*some, causal=True).square().sum(), [some[n]])
        assert torch.equal(got, want[n])
    x = q.clone().requires_grad_(True)
    y = tv.attention(x, x[:, :, :2], x[:, :, 2:], causal=True)        # one leaf as all three operands
    (got,) = torch.autograd.grad(y.square().sum(), x)
    parts = [q.clone().requires_grad_(True), q[:, :, :2].clone().requires_grad_(True), q[:, :, 2:].clone().requires_grad_(True)]
    dq, dk, dv = torch.autograd.grad(tv.attention(*parts, causal=True).square().sum(), parts)
    assert torch.allclose(got, dq + torch.cat([dk, dv], 2), rtol=1e-6, atol=1e-6)
    y = tv.attention(x, k, v)
    with pytest.raises(RuntimeError):                                    # a saved operand changed in place
        k.add_(1.0)
        y.sum().backward()
    with pytest.raises(RuntimeError):                                    # no second derivatives
        z = tv.attention(x, k, v)
        (gx,) = torch.autograd.grad(z.square().sum(), x, create_graph=True)
        gx.sum().backward()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_infinities_and_nan_behind_a_mask_stay_there(tv, dev, kind, bad):
    """Documents 0 | 1 | padding; everything that belongs to document 1 and to the padding is spoiled: document 0 keeps its bits, results and
    gradients.  The same for keys that no query sees."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(31)
    b, t, hq, hk, d = 1, 200, 4, 2, 64
    ids = torch.where(torch.arange(t) < 90, 0, torch.where(torch.arange(t) < 170, 1, -1))[None]
    clean = [normal(g, b, t, h, d, dtype=dt) for h in (hq, hk, hk, hq)]
    for causal in (True, False):
        results = []
        for spoil in (False, True):
            x = [y.clone() for y in clean]
            if spoil:
                for y in x:
                    y[:, 90:, :, ::3] = bad
                    y[:, 95] = bad
            leaves = [y.to(dev).requires_grad_(True) for y in x[:3]]
            out = tv.attention(*leaves, causal=causal, documents=ids.to(dev))
            results.append([out[:, :90]] + [y[:, :90] for y in torch.autograd.grad(out, leaves, x[3].to(dev))])
        for x, y in zip(*results):
            assert torch.equal(x, y)
    # causal: a spoiled last token (its query, key, value and gradient) spoils its own row and the gradients it takes part in, nothing in front of it
    x = [y.clone() for y in clean]
    x[1][:, -1] = bad
    x[2][:, -1] = bad
    leaves = [y.to(dev).requires_grad_(True) for y in x[:3]]
    out = tv.attention(*leaves, causal=True)
    ref = tv.attention(*[y.to(dev) for y in clean[:3]], causal=True)
    assert torch.equal(out[:, :-1], ref[:, :-1]) and not torch.isfinite(out[:, -1].float()).any()
    go = x[3].to(dev).clone()
    go[:, -1] = 0
    leaves0 = [y.to(dev).requires_grad_(True) for y in clean[:3]]
    want = torch.autograd.grad(tv.attention(*leaves0, causal=True), leaves0, go)
    got = torch.autograd.grad(out, leaves, go)
    assert torch.equal(got[0][:, :-1], want[0][:, :-1])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_infinities_behind_a_prefix_that_ends_inside_a_tile(tv, dev, kind, bad):
    """Queries that all see the same prefix, with spoiled keys behind it in the same tile: they keep their bits, results and gradients."""
    g = torch.Generator().manual_seed(37)
    for d, t, prefix, at in ((64, 190, 70, 100), (128, 190, 70, 71), (64, 330, 230, 240)):
        clean = [normal(g, 2, t, h, d, dtype=TYPES[kind]) for h in (4, 2, 2, 4)]
        results = []
        for spoil in (False, True):
            x = [y.clone() for y in clean]
            if spoil:
                x[1][:, at:] = bad
                x[2][:, at:] = bad
            leaves = [y.to(dev).requires_grad_(True) for y in x[:3]]
            out = tv.attention(*leaves, causal=True, prefix=prefix)
            (dq,) = torch.autograd.grad(out, leaves[0], x[3].to(dev))
            with torch.no_grad():
                cached = tv.cached_attention(leaves[0], *(y.transpose(1, 2).contiguous() for y in leaves[1:]), 0, prefix=prefix)
            results.append([out[:, :at], dq[:, :at], cached[:, :at]])
        for x, y, name in zip(*results, ("out", "dq", "cached")):
            assert torch.equal(x, y), (name, d)


def test_attention_visible_infinities_show(tv, dev):
    """A value of +-infinity that a query sees gives that infinity (NaN for both signs), at its element alone."""
    q, k, v = (torch.randn(1, 40, 1, 64, device=dev) for _ in range(3))
    v[0, 3, 0, 5], v[0, 6, 0, 5], v[0, 8, 0, 7] = math.inf, -math.inf, math.nan
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        out = tv.attention(q.to(dt), k.to(dt), v.to(dt), causal=True)[0, :, 0].float()
        assert torch.isfinite(out[:3]).all() and (out[3:6, 5] == math.inf).all() and torch.isnan(out[6:, 5]).all() and torch.isnan(out[8:, 7]).all()
        rest = out.clone()
        rest[:, [5, 7]] = 0
        assert torch.isfinite(rest).all()
    k[0, 2] = math.nan
    out = tv.attention(q, k, v, causal=True)[0, :, 0]
    assert torch.isfinite(out[:2]).all() and torch.isnan(out[2:]).all()


def test_attention_refusals(tv, dev):
    q, k = torch.randn(2, 5, 4, 64, device=dev), torch.randn(2, 5, 2, 64, device=dev)
    ids = torch.zeros(2, 5, dtype=torch.int64, device=dev)
    cases = [lambda: tv.attention(q, k, k[:, :4]), lambda: tv.attention(q, k.half(), k.half()), lambda: tv.attention(q[:, :, :3], k, k), lambda: tv.attention(q, k[..., :32], k[..., :32]),
             lambda: tv.attention(torch.randn(2, 5, 4, 129, device=dev), torch.randn(2, 5, 4, 129, device=dev), torch.randn(2, 5, 4, 129, device=dev)),
             lambda: tv.attention(q, k, k, scale=math.nan), lambda: tv.attention(q, k, k, softcap=-1.0), lambda: tv.attention(q, k, k, slopes=torch.ones(3, device=dev)),
             lambda: tv.attention(q, k, k, slopes=torch.ones(4, device=dev, requires_grad=True)), lambda: tv.attention(q, k, k, slopes=torch.ones(4)),
             lambda: tv.attention(q, k, k, prefix=3), lambda: tv.attention(q, k, k, causal=True, prefix=torch.zeros(2, device=dev)),
             lambda: tv.attention(q, k, k, documents=ids.int()), lambda: tv.attention(q, k[:, :4], k[:, :4], documents=ids), lambda: tv.attention(q, k, k, documents=ids[:, :4]),
             lambda: tv.attention(q[0], k[0], k[0]), lambda: tv.attention(q.double(), k.double(), k.double()), lambda: tv.attention(q[:, :, :0], k, k), lambda: tv.attention(q.cpu(), k, k),
             lambda: tv.attention(q[..., :0], k[..., :0], k[..., :0])]
    for n, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {n} was not refused")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("documents", [False, True])
def test_calls_stay_inside_the_workspace_they_ask_for(tv, dev, kind, documents, monkeypatch):
    """Every workspace is handed out with a margin of known bytes on both sides, which have to be there afterwards."""
    A = tv.attention_ops
    given = []

    def workspace(need, device):
        if need == 0:
            return None, 0
        ws = torch.full((need + 2 * 65536,), 0xA5, dtype=torch.uint8, device=device)
        given.append((ws, need))
        return ws, ws.data_ptr() + 65536

    monkeypatch.setattr(A, "_workspace", workspace)
    dt = TYPES[kind]
    for b, t, h, hk, d in ((3, 130, 4, 2, 64), (1, 1, 1, 1, 64), (2, 700, 2, 1, 128)):
        leaves = [torch.randn(b, t, n, d, device=dev, dtype=dt, requires_grad=True) for n in (h, hk, hk)]
        ids = (torch.arange(t, device=dev) // 50)[None].repeat(b, 1) if documents else None
        out = tv.attention(*leaves, causal=True, documents=ids)
        torch.autograd.grad(out, leaves, torch.randn_like(out))
        with torch.no_grad():
            for n in (1, min(t, 4), t):
                tv.cached_attention(leaves[0][:, :n].detach(), leaves[1].detach().transpose(1, 2), leaves[2].detach().transpose(1, 2), t - n)
                long = torch.randn(2, hk, 9000, d, device=dev, dtype=dt)
                tv.cached_attention(torch.randn(2, n, h, d, device=dev, dtype=dt), long, long, 8000)
    torch.cuda.synchronize()
    assert given
    for ws, need in given:
        assert bool((ws[:65536] == 0xA5).all()) and bool((ws[65536 + need:] == 0xA5).all()), need


def test_attention_empty_calls(tv, dev):
    z = lambda *s: torch.randn(*s, device=dev, requires_grad=True)
    for b, tq, tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0), (2, 0, 0)):
        leaves = [z(b, tq, 4, 64), z(b, tk, 2, 64), z(b, tk, 2, 64)]
        out = tv.attention(*leaves, causal=True)
        assert out.shape == (b, tq, 4, 64) and int(out.count_nonzero()) == 0
        for x, y in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
            assert x.shape == y.shape and int(x.count_nonzero()) == 0


def test_attention_on_another_stream_and_captured(tv, dev):
    """Forward and backward on a side stream, and as a captured graph replayed with new contents between eager calls on the same leaves."""
    g = torch.Generator().manual_seed(41)
    leaves = [normal(g, 2, 150, h, 64, dtype=torch.float16).to(dev).requires_grad_(True) for h in (4, 2, 2)]
    go = normal(g, 2, 150, 4, 64, dtype=torch.float16).to(dev)
    table = tv.rotary_table(32, 150, device=dev)
    pos = torch.arange(150, device=dev)

    def step():
        q, k, v = leaves
        out = tv.attention(tv.rotary(q, pos, table), tv.rotary(k, pos, table), v, causal=True, softcap=10.0)
        return [out] + list(torch.autograd.grad(out, leaves, go))

    eager = [x.detach().clone() for x in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = [x.detach() for x in step()]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(eager, side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        static = step()
    for n in range(3):
        with torch.no_grad():
            for x in leaves:
                x.copy_(normal(g, *x.shape, dtype=torch.float16).to(dev))
        want = [x.detach().clone() for x in step()]                       # eager work between the replays
        torch.cuda.synchronize()
        graph.replay()
        junk = torch.full((1 << 22,), float("nan"), device=dev)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, static)), n
        del junk


def test_capture_beside_a_live_eager_graph_is_refused(tv, dev):
    """The gradient node of a leaf belongs to the stream of the eager call that made it: recording a backward pass over it would end the
    process.  The call is refused; once the eager result is gone the capture works."""
    q, k, v = (torch.randn(1, 20, 2, 64, device=dev, requires_grad=True) for _ in range(3))
    table, pos, go = tv.rotary_table(32, 20, device=dev), torch.arange(20, device=dev), torch.randn(1, 20, 2, 64, device=dev)
    for call in (lambda: tv.attention(q, k, v), lambda: tv.rotary(q, pos, table)):
        alive = call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph, stream=s):
                call()
        want = alive.detach().clone()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
            (gq,) = torch.autograd.grad(out, q, go)
        for _ in range(2):
            out.detach().zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del out, gq, graph


# ---------------------------------------------------------------------------------------------------- cached attention

def run_cached(tv, dev, kind, b, t, hq, hk, d, slots, lens, prefix=None, count=None, softcap=0.0, slopes=False, scale=None, seed=0, spoil=True):
    g = torch.Generator().manual_seed(seed + t + slots + d)
    dt = TYPES[kind]
    q, kc, vc = normal(g, b, t, hq, d, dtype=dt), normal(g, b, hk, slots, d, dtype=dt), normal(g, b, hk, slots, d, dtype=dt)
    sl = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)]) if slopes else None
    lens = torch.as_tensor(lens)
    n = torch.full((b,), t) if count is None else torch.as_tensor(count)
    pre = torch.zeros(b, dtype=torch.int64) if prefix is None else (torch.full((b,), prefix) if isinstance(prefix, int) else torch.as_tensor(prefix))
    see, place = R.sees(b, t, slots, True, pre, None, lens.expand(b) if lens.dim() == 0 else lens, n)
    ref = R.Attention(q, kc.transpose(1, 2), vc.transpose(1, 2), see, place, scale, softcap, sl)
    if spoil:                                                              # what lies behind the filled part is never used
        for i in range(b):
            end = int((lens if lens.dim() == 0 else lens[i]) + n[i])
            kc[i, :, end:] = math.nan
            vc[i, :, end:] = math.inf
    on = lambda x: x.to(dev) if isinstance(x, torch.Tensor) else x
    args = (q.to(dev), kc.to(dev), vc.to(dev), lens.to(dev))
    kw = dict(scale=scale, softcap=softcap, slopes=on(sl), prefix=None if prefix is None else (prefix if isinstance(prefix, int) else pre.to(dev)),
              count=None if count is None else n.to(dev))
    out = tv.cached_attention(*args, **kw)
    R.within(out, *ref.forward(), what="cached")
    assert torch.equal(out, tv.cached_attention(*args, **kw))
    return out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("b,t,hq,hk,d,slots,lens", [
    (1, 1, 4, 4, 64, 64, 0), (1, 1, 32, 32, 64, 1024, 745), (3, 1, 8, 2, 64, 300, [0, 17, 299]), (2, 1, 8, 1, 128, 2000, [1999, 1000]), (1, 1, 16, 1, 64, 5000, 4999),
    (2, 1, 32, 1, 64, 200, [100, 199]), (2, 3, 4, 2, 64, 130, [0, 120]), (1, 8, 4, 1, 128, 700, 600), (2, 20, 4, 2, 64, 300, [0, 250]), (1, 70, 2, 2, 64, 200, 130), (2, 150, 4, 2, 96, 400, [0, 250]),
    (1, 5, 2, 1, 33, 50, 7), (2, 1, 3, 3, 80, 90, [3, 89]), (1, 1, 1, 1, 1, 1, 0), (1, 1, 4, 2, 64, 9000, 8999)])
def test_cached_attention_shapes(tv, dev, kind, b, t, hq, hk, d, slots, lens):
    run_cached(tv, dev, kind, b, t, hq, hk, d, slots, lens)
    run_cached(tv, dev, kind, b, t, hq, hk, d, slots, lens, softcap=4.0, slopes=True, scale=0.2, seed=1)


@pytest.mark.parametrize("kind", TYPES)
def test_cached_attention_prefix_and_counts(tv, dev, kind):
    run_cached(tv, dev, kind, 4, 9, 4, 2, 64, 60, [0, 5, 40, 51], prefix=[0, 3, 60, 100], count=[9, 0, 4, 1], seed=2)
    run_cached(tv, dev, kind, 2, 130, 4, 4, 64, 200, [0, 0], prefix=100, count=[130, 77], seed=3)
    run_cached(tv, dev, kind, 2, 1, 8, 2, 128, 1500, [1400, 3], prefix=1300, seed=3)
    out = run_cached(tv, dev, kind, 3, 40, 2, 1, 64, 100, [10, 0, 60], count=[7, 0, 40], seed=4)
    assert int(out[0, 7:].count_nonzero()) == 0 and int(out[1].count_nonzero()) == 0


def test_cached_attention_bad_lengths_and_refusals(tv, dev):
    q = torch.randn(4, 3, 4, 64, device=dev)
    k, v = (torch.randn(4, 2, 10, 64, device=dev) for _ in range(2))
    lens = torch.tensor([-1, 8, 1 << 62, -(1 << 62)], device=dev)
    out = tv.cached_attention(q, k, v, lens)
    assert torch.isnan(out[[0, 2, 3]]).all() and torch.isfinite(out[1, :2]).all() and torch.isnan(out[1, 2]).all()
    one = tv.cached_attention(q[:, :1], k, v, torch.tensor([-1, 9, 10, 1 << 62], device=dev))
    assert torch.isnan(one[[0, 2, 3]]).all() and torch.isfinite(one[1]).all()
    odd = torch.tensor([-3, 100, 1, 3], device=dev)                            # counts are clamped to [0, tokens]
    got = tv.cached_attention(q, k, v, 2, count=odd)
    assert torch.equal(got, tv.cached_attention(q, k, v, 2, count=odd.clamp(0, 3)))
    assert tv.cached_attention(q[:, :0], k, v, 0).shape == (4, 0, 4, 64) and tv.cached_attention(q[:0], k[:0], v[:0], 0).shape == (0, 3, 4, 64)
    cases = [lambda: tv.cached_attention(q, k, v, 8), lambda: tv.cached_attention(q, k, v, -1), lambda: tv.cached_attention(q, k, v[:, :, :9], 0), lambda: tv.cached_attention(q, k.half(), v.half(), 0),
             lambda: tv.cached_attention(q[:, :, :3], k, v, 0), lambda: tv.cached_attention(q, k, v, lens.int()), lambda: tv.cached_attention(q, k, v, lens[:3]),
             lambda: tv.cached_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, 0), lambda: tv.cached_attention(q, k, v, 0, count=lens[:3]),
             lambda: tv.cached_attention(q.clone().requires_grad_(True), k, v, 0), lambda: tv.cached_attention(q[:2], k, v, 0), lambda: tv.cached_attention(q, k, v, 0, softcap=math.inf)]
    for n, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {n} was not refused")


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_cached_attention_later_tokens_of_a_chunk_do_not_reach_earlier_ones(tv, dev, kind, bad):
    g = torch.Generator().manual_seed(51)
    dt = TYPES[kind]
    for t, hq, hk in ((4, 4, 2), (80, 2, 2)):
        q, k, v = normal(g, 1, t, hq, 64, dtype=dt).to(dev), normal(g, 1, hk, 200, 64, dtype=dt).to(dev), normal(g, 1, hk, 200, 64, dtype=dt).to(dev)
        want = tv.cached_attention(q, k, v, 70)
        k[:, :, 70 + t - 1:], v[:, :, 70 + t - 1:] = bad, bad
        got = tv.cached_attention(q, k, v, 70)
        assert torch.equal(got[:, :-1], want[:, :-1]) and not torch.isfinite(got[:, -1].float()).any()


def test_cached_attention_offsets_beyond_32_bits(tv, dev):
    """Caches of more than 2^32 elements: the last sequence's and the last slots' rows lie past 32-bit offsets."""
    slots, d = 17_000_000, 128
    k, v = (torch.empty((2, 1, slots, d), dtype=torch.float16, device=dev) for _ in range(2))
    assert k.numel() > 1 << 32
    g = torch.Generator().manual_seed(61)
    q, kn, vn = normal(g, 2, 1, 2, d, dtype=torch.float16).to(dev), normal(g, 2, 1, 90, d, dtype=torch.float16).to(dev), normal(g, 2, 1, 90, d, dtype=torch.float16).to(dev)
    k[:, :, :90], v[:, :, :90] = kn, vn
    lens = torch.tensor([50, 89], device=dev)
    assert torch.equal(tv.cached_attention(q, k, v, lens), tv.cached_attention(q, kn.contiguous(), vn.contiguous(), lens))
    # slots far apart: the cache of one sequence as every 100000th row of the big one
    ks, vs = k[1:, :, ::100_000], v[1:, :, ::100_000]
    kd, vd = normal(g, 1, 1, 170, d, dtype=torch.float16).to(dev), normal(g, 1, 1, 170, d, dtype=torch.float16).to(dev)
    ks.copy_(kd), vs.copy_(vd)
    at = torch.tensor([168], device=dev)
    assert torch.equal(tv.cached_attention(q[:1], ks, vs, at), tv.cached_attention(q[:1], kd, vd, at))
    table = tv.rotary_table(32, 170, device=dev)
    qkv = normal(g, 1, 1, 4 * d, dtype=torch.float16).to(dev)
    assert torch.equal(tv.rotary_cache(qkv, table, ks, vs, at, 2), tv.rotary_cache(qkv, table, kd, vd, at, 2))
    assert torch.equal(ks[:, :, 168], kd[:, :, 168]) and torch.equal(vs[:, :, 168], vd[:, :, 168])
    del k, v, ks, vs
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------------ a run of them

@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hq,hk,softcap,slopes", [(4, 4, 0.0, False), (8, 2, 20.0, True)])
def test_serving_forms_continue_what_the_training_forms_compute(tv, dev, kind, hq, hk, softcap, slopes):
    """A prompt, a chunk and single tokens through rotary_cache + cached_attention give each token what rotary + attention give it
    over the whole sequence at once."""
    g = torch.Generator().manual_seed(71)
    dt, d, total, b = TYPES[kind], 64, 90, 2
    qkv = normal(g, b, total, (hq + 2 * hk) * d, dtype=dt).to(dev)
    table = tv.rotary_table(32, 128, device=dev)
    sl = torch.tensor([2.0 ** -(i + 1) for i in range(hq)], device=dev) if slopes else None
    heads = qkv.unflatten(-1, (hq + 2 * hk, d))
    both = tv.rotary(heads[:, :, : hq + hk], torch.arange(total, device=dev), table)
    whole = tv.attention(both[:, :, :hq], both[:, :, hq:], heads[:, :, hq + hk:], causal=True, softcap=softcap, slopes=sl, prefix=21)
    k, v = (torch.full((b, hk, 128, d), math.nan, dtype=dt, device=dev) for _ in range(2))
    lens, outs, at = torch.zeros((), dtype=torch.int64, device=dev), [], 0
    for n in (60, 7, 1, 1, 20, 1):
        q = tv.rotary_cache(qkv[:, at: at + n], table, k, v, lens, hq)
        assert torch.equal(q, both[:, at: at + n, :hq])
        outs.append(tv.cached_attention(q, k, v, lens, softcap=softcap, slopes=sl, prefix=21))
        at += n
        lens += n
    assert torch.equal(k[:, :, :total].transpose(1, 2), both[:, :, hq:]) and torch.isnan(k[:, :, total:].float()).all()
    see, place = R.sees(b, total, total, True, torch.full((b,), 21), None)
    c = lambda x: x.cpu()
    ref = R.Attention(c(both[:, :, :hq]), c(both[:, :, hq:]), c(heads[:, :, hq + hk:]), see, place, None, softcap, None if sl is None else sl.cpu())
    R.within(whole, *ref.forward(), what="whole")
    R.within(torch.cat(outs, 1), *ref.forward(), what="pieces")


def test_decode_step_captured_and_replayed(tv, dev):
    """rotary_cache and cached_attention in one graph with the fill level on the device: every replay advances, eager work between the replays."""
    g = torch.Generator().manual_seed(81)
    b, hq, hk, d, slots = 2, 8, 2, 64, 400
    table = tv.rotary_table(d, slots, device=dev)
    k, v = (normal(g, b, hk, slots, d, dtype=torch.float16).to(dev) for _ in range(2))
    lens = torch.tensor([5, 380], device=dev)
    x = torch.zeros(b, 1, (hq + 2 * hk) * d, dtype=torch.float16, device=dev)

    def step(k, v, lens):
        q = tv.rotary_cache(x, table, k, v, lens, hq)
        return tv.cached_attention(q, k, v, lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(k.clone(), v.clone(), lens)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k, v, lens)
        lens += 1
    k2, v2, lens2 = k.clone(), v.clone(), lens.clone()
    for n in range(6):
        x.copy_(normal(g, *x.shape, dtype=torch.float16).to(dev))
        want = step(k2, v2, lens2)
        lens2 += 1
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lens, lens2), n
    assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("fused_product", [True, False])
def test_decode_harness_with_fused_attention(tv, dev, fused_product):
    """The decoder stack with rotary_cache + cached_attention against the same stack with the tensor operations (float32: both evaluate the same sums to
    about 1e-6 an operation; the bound is that of packed against dense products), and its captured step against the eager one bit for bit."""
    from ternary_vllm_amd import decode_harness as dh
    kw = dict(hidden=256, heads=4, intermediate=1024, blocks=2, max_len=64, fuse_qkv_fc1=fused_product)
    torch.manual_seed(3)
    prompt = torch.randn(2, 19, 256, device=dev)
    toks = [torch.randn(2, 1, 256, device=dev) for _ in range(4)]

    def run(fuse, graph):
        st = dh.TernaryDecoderStack(dh.DecoderConfig(fuse_attention=fuse, **kw), batch=2, device=dev, dtype=torch.float32, seed=11)
        with torch.no_grad():
            outs = [st.prefill(prompt)]
            if graph:
                st.capture_decode(toks[0])
            outs += [(st.decode_graph(t) if graph else st.decode_step(t)).clone() for t in toks]
        assert int(st.pos) == 19 + len(toks)
        return outs

    plain, fused, replay = run(False, False), run(True, False), run(True, True)
    for a, b in zip(fused, plain):
        assert a.shape == b.shape and float((a - b).abs().max()) <= 2e-4 * max(1.0, float(b.abs().max()))
    for a, b in zip(fused, replay):
        assert torch.equal(a, b)
