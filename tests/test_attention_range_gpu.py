"""Attention where numbers of very different size meet: score gradients of large values, of losses that differ by many powers of ten between documents,
tokens and queries; rows of many small weights, caps far above the scores: against float64 within the bounds of tests/attention_bounds.py."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attention_reference as R  # noqa: E402
from attention_bounds import Tight  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tv():
    import ternary_vllm_amd
    return ternary_vllm_amd


def normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def within(got, want, tol, what):
    """R.within; where the exact value may lie beyond the type's largest one, the infinity of its sign is a rounding of it."""
    got, want = got.detach().cpu(), want.to(torch.float64)
    beyond = (want.abs() + tol >= torch.finfo(got.dtype).max) & (got == torch.copysign(torch.full_like(want, math.inf), want))
    R.within(torch.where(beyond, want, got.double()), want, tol, what)


def run_training(tv, dev, q, k, v, go, causal=False, documents=None, softcap=0.0, prefix=None, scale=None, slopes=None):
    """Result and gradients within Tight's bounds; returns them."""
    b, tq, tk = q.shape[0], q.shape[1], k.shape[1]
    see, place = R.sees(b, tq, tk, causal, torch.full((b,), prefix or 0), documents)
    ref = Tight(q, k, v, see, place, scale, softcap, slopes)
    leaves = [x.clone().to(dev).requires_grad_(True) for x in (q, k, v)]
    out = tv.attention(*leaves, causal=causal, softcap=softcap, prefix=prefix, scale=scale, slopes=None if slopes is None else slopes.to(dev), documents=None if documents is None else documents.to(dev))
    within(out, *ref.forward(), what="out")
    grads = torch.autograd.grad(out, leaves, go.to(dev))
    for name, got, (want, tol) in zip(("dq", "dk", "dv"), grads, ref.grads(go)):
        within(got, want, tol, name)
    return [out.detach(), *grads]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value,gradient", [(70.0, 0.0624), (3000.0, 0.0624), (70.0, 15.0), (60000.0, 0.001)])
def test_score_gradients_of_large_values(tv, dev, kind, d, value, gradient):
    """Rows of values of one sign against output gradients of one sign: their products, far beyond float16's range here and there, belong to gradients that are not."""
    dt = TYPES[kind]
    # one query, two keys of equal score: dq = scale * gradient * value * d * (k0 - k1) / 2 * 2 / 2
    q, go = torch.zeros(1, 1, 1, d, dtype=dt), torch.full((1, 1, 1, d), gradient, dtype=dt)
    k, v = torch.zeros(1, 2, 1, d, dtype=dt), torch.full((1, 2, 1, d), value, dtype=dt)
    q[..., 1] = 1.0                                     # apart from the keys: the scores stay 0
    k[:, 0, :, 0], k[:, 1, :, 0] = 0.25, -0.25
    v[:, 1] = -v[:, 1]
    want = d ** -0.5 * float(go[0, 0, 0, 0]) * float(v[0, 0, 0, 0]) * d * 0.25
    _, dq, dk, _ = run_training(tv, dev, q, k, v, go)
    assert abs(float(dq[0, 0, 0, 0]) - want) <= 2.0 ** -7 * want and abs(float(dk[0, 0, 0, 1]) - 2 * want) <= 2.0 ** -7 * 2 * want
    g = torch.Generator().manual_seed(d)
    t = 150
    sign = torch.where(torch.rand(1, t, 2, 1, generator=g) < 0.5, -1.0, 1.0)
    q, k = normal(g, 1, t, 4, d, dtype=dt, scale=0.01), normal(g, 1, t, 2, d, dtype=dt, scale=0.01)
    v = (sign * value * (1 + 0.02 * torch.randn(1, t, 2, d, generator=g))).to(dt)
    go = (gradient * (1 + 0.02 * torch.randn(1, t, 4, d, generator=g))).to(dt)
    run_training(tv, dev, q, k, v, go, causal=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("small,large", [(0.01, 15.0), (1e-4, 100.0), (0.02, 30000.0)])
def test_documents_of_different_losses(tv, dev, kind, d, causal, small, large):
    """A document's gradients have the accuracy they have alone, beside documents of much larger ones, and the same bits."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(91 + d)
    t = 260
    ids = torch.where(torch.arange(t) < 100, 0, torch.where(torch.arange(t) < 230, 1, 2))[None]
    q, k, v, go = (normal(g, 1, t, h, d, dtype=dt, scale=s) for h, s in ((4, 1.0), (2, 1.0), (2, 1.0), (4, small)))
    loud = go.clone()
    loud[:, 100:230] = (torch.rand(1, 130, 4, d, generator=g) * large).to(dt)
    alone = run_training(tv, dev, q, k, v, go, causal, ids)
    beside = run_training(tv, dev, q, k, v, loud, causal, ids)
    for x, y in zip(alone, beside):
        assert torch.equal(x[:, :100], y[:, :100]) and torch.equal(x[:, 230:], y[:, 230:])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("large", [100.0, 30000.0])
def test_a_large_gradient_at_a_token_that_others_do_not_see(tv, dev, kind, d, large):
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(95 + d)
    t = 400
    q, k, v, go = (normal(g, 1, t, h, d, dtype=dt, scale=s) for h, s in ((2, 1.0), (1, 1.0), (1, 1.0), (2, 0.02)))
    loud = go.clone()
    loud[:, 0, :, 0] = large                             # the first query sees the first key alone
    alone, beside = run_training(tv, dev, q, k, v, go, True), run_training(tv, dev, q, k, v, loud, True)
    assert torch.equal(alone[2][:, 1:], beside[2][:, 1:]) and torch.equal(alone[1][:, 1:], beside[1][:, 1:])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_gradients_of_every_size_at_once(tv, dev, kind, softcap):
    """Queries whose output gradients differ by powers of ten from token to token, in rising, falling and mixed order."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(97)
    for order in (torch.arange(200), torch.arange(199, -1, -1), torch.randperm(200, generator=g)):
        size = 10.0 ** (order.double() / 199 * 8 - 6)     # 1e-6 .. 1e2
        q, k, v, go = (normal(g, 1, 200, h, 64) for h in (2, 2, 2, 2))
        go = go * size[None, :, None, None].float()
        run_training(tv, dev, *(x.to(dt) for x in (q, k, v, go)), causal=False, softcap=softcap)
        run_training(tv, dev, *(x.to(dt) for x in (q, k, v, go)), causal=True, softcap=softcap)


def small_weights(kind, d, queries, keys, away):
    """One key of value 0 and score 0, all others of value 1 and a score of -away * ln 2: scale 1, the first element of a head carries the score."""
    dt = TYPES[kind]
    q, k, v = torch.zeros(1, queries, 2, d, dtype=dt), torch.zeros(1, keys, 1, d, dtype=dt), torch.ones(1, keys, 1, d, dtype=dt)
    q[..., 0] = 1.0
    k[..., 0] = -away * math.log(2.0)
    return q, k, v


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("away", [24.5, 25.2, 28.0, 31.0])
def test_many_small_weights_count(tv, dev, kind, d, away):
    """Weights far below the largest one of their row: together they are a result."""
    q, k, v = small_weights(kind, d, 40, 20000, away)
    for top in (0, 7000, 19999):                         # where the large score is: the running maximum finds it early or late
        kt, vt = k.clone(), v.clone()
        kt[:, top, :, 0], vt[:, top] = 0.0, 0.0
        see, place = R.sees(1, 40, 20000, False, torch.zeros(1, dtype=torch.int64), None)
        want, tol = Tight(q, kt, vt, see, place, 1.0).forward()
        # whole rows, a few tokens over a cache (cut into parts), many tokens over a cache
        within(tv.attention(q.to(dev), kt.to(dev), vt.to(dev), scale=1.0), want, tol, "attention")
        if top == 19999:
            continue                                     # only the last token of a chunk would see it
        cache = [x.transpose(1, 2).contiguous().to(dev) for x in (kt, vt)]
        for n in (1, 8, 40):
            at = 20000 - n
            see, place = R.sees(1, n, 20000, True, torch.zeros(1, dtype=torch.int64), None, torch.tensor([at]), torch.tensor([n]))
            want, tol = Tight(q[:, :n], kt, vt, see, place, 1.0).forward()
            within(tv.cached_attention(q[:, :n].to(dev), *cache, at, scale=1.0), want, tol, f"cached {n}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("away", [24.5, 25.2, 28.0, 31.0])
def test_value_gradients_of_many_small_weights(tv, dev, kind, d, away):
    q, k, v = small_weights(kind, d, 700, 200, away)
    k[:, 3, :, 0] = 0.0
    go = torch.ones(1, 700, 2, d, dtype=TYPES[kind]) * 50
    run_training(tv, dev, q, k, v, go, scale=1.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("softcap", [64.0, 65.0, 1e3, 1e5, 1e7])
@pytest.mark.parametrize("d", [64, 128])
def test_caps_far_above_the_scores(tv, dev, kind, softcap, d):
    """A cap bends the scores near it and leaves the others alone, whatever its size."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(101 + d)
    for spread, slopes in ((1.0, None), (8.0, torch.tensor([0.5, 0.01, 0.0, 0.1]))):
        q, k, v, go = (normal(g, 2, 110, h, d, dtype=dt, scale=s) for h, s in ((4, spread), (2, 1.0), (2, 1.0), (4, 0.02)))
        run_training(tv, dev, q, k, v, go, causal=True, softcap=softcap, slopes=slopes)
        see, place = R.sees(2, 3, 110, True, torch.zeros(2, dtype=torch.int64), None, torch.tensor([107, 40]), torch.tensor([3, 3]))
        want, tol = Tight(q[:, :3], k, v, see, place, None, softcap, slopes).forward()
        cache = [x.transpose(1, 2).contiguous().to(dev) for x in (k, v)]
        within(tv.cached_attention(q[:, :3].to(dev), *cache, torch.tensor([107, 40], device=dev), softcap=softcap, slopes=None if slopes is None else slopes.to(dev)), want, tol, "cached")
    # scores near and beyond the cap
    q, k, v, go = (normal(g, 1, 60, h, d, dtype=dt, scale=s) for h, s in ((2, softcap ** 0.5 if softcap <= 1e5 else 1.0), (2, softcap ** 0.5 if softcap <= 1e5 else 1.0), (2, 1.0), (2, 0.02)))
    run_training(tv, dev, q, k, v, go, causal=True, softcap=softcap)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("softcap", [2.0 ** 100, 1e38, 3.4e38])
def test_caps_at_the_end_of_float32(tv, dev, kind, softcap):
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(103)
    q, k, v, go = (normal(g, 1, 70, h, 64, dtype=dt, scale=s) for h, s in ((4, 1.0), (2, 1.0), (2, 1.0), (4, 0.02)))
    run_training(tv, dev, q, k, v, go, causal=True, softcap=softcap)
    cache = [x.transpose(1, 2).contiguous().to(dev) for x in (k, v)]
    for n in (1, 70):
        see, place = R.sees(1, n, 70, True, torch.zeros(1, dtype=torch.int64), None, torch.tensor([70 - n]), torch.tensor([n]))
        want, tol = Tight(q[:, :n], k, v, see, place, None, softcap).forward()
        within(tv.cached_attention(q[:, :n].to(dev), *cache, 70 - n, softcap=softcap), want, tol, f"cached {n}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,causal,softcap", [(30, 2, True, 0.0), (30, 2, False, 4.0), (9, 3, True, 0.0), (4, 16, True, 3.0), (3, 65, False, 0.0), (2, 127, True, 0.0), (2, 127, False, 0.0)])
def test_gradients_of_few_keys_keep_their_digits(tv, dev, kind, d, b, t, causal, softcap):
    """Where a query sees few keys, the rounding of its result would be as large in its gradients as their own."""
    g = torch.Generator().manual_seed(109 + t)
    q, k, v, go = (normal(g, b, t, h, d, dtype=TYPES[kind], scale=s) for h, s in ((4, 1.0), (2, 1.0), (2, 1.0), (4, 0.02)))
    _, dq, dk, dv = run_training(tv, dev, q, k, v, go, causal=causal, softcap=softcap)
    for wanted in ((0,), (1,), (2,), (0, 2)):            # a gradient does not depend on which others are wanted
        leaves = [x.clone().to(dev).requires_grad_(n in wanted) for n, x in enumerate((q, k, v))]
        got = torch.autograd.grad(tv.attention(*leaves, causal=causal, softcap=softcap), [leaves[n] for n in wanted], go.to(dev))
        assert all(torch.equal(x, (dq, dk, dv)[n]) for n, x in zip(wanted, got))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_short_documents_keep_their_digits(tv, dev, kind, causal):
    """Documents of 1 to 90 tokens, in runs and interleaved, some padding between them."""
    g = torch.Generator().manual_seed(113)
    ids = torch.tensor(sum([[n] * s for n, s in enumerate((1, 2, 3, 60, 90, 5, 40, 64, 35))], []))
    ids[70:74] = -1
    for docs in (ids, torch.arange(300) % 7):
        q, k, v, go = (normal(g, 1, 300, h, 64, dtype=TYPES[kind], scale=s) for h, s in ((2, 1.0), (2, 1.0), (2, 1.0), (2, 0.02)))
        run_training(tv, dev, q, k, v, go, causal=causal, documents=docs[None])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_gradients_of_rows_whose_weight_lies_on_few_keys(tv, dev, kind, d, softcap):
    """Long rows that a steep bias or large scores leave a few keys of."""
    g = torch.Generator().manual_seed(127 + d)
    for spread, slopes in ((0.5, torch.tensor([2.0, 1.0, 0.5, 0.25])), (4.0, None)):
        q, k, v, go = (normal(g, 1, 400, h, d, dtype=TYPES[kind], scale=s) for h, s in ((4, spread), (2, 1.0), (2, 1.0), (4, 0.02)))
        run_training(tv, dev, q, k, v, go, causal=True, softcap=softcap, slopes=slopes)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("softcap,slopes", [(0.0, False), (6.0, True)])
def test_queries_of_one_key_have_no_score_gradient(tv, dev, kind, softcap, slopes):
    """A softmax over one key is 1 whatever its score: zeros, not the rounding of a difference."""
    g = torch.Generator().manual_seed(131)
    sl = torch.tensor([0.5, 0.1, 0.01, 1.0]) if slopes else None
    for b, tq, tk, causal, d in ((9, 1, 1, True, 64), (3, 1, 1, False, 128), (2, 70, 1, False, 64), (2, 150, 20, True, 64), (1, 40, 40, True, 33), (2, 300, 300, True, 128)):
        q, k, v, go = (normal(g, b, t, h, d, dtype=TYPES[kind]) for t, h in ((tq, 4), (tk, 2), (tk, 2), (tq, 4)))
        first = max(0, tq - tk) if causal else tq - 1                    # the last query that sees one key at most
        if causal or tk == 1:
            only = go.clone()
            only[:, first + 1:] = 0                                      # gradients of those queries alone
            _, dq, dk, _ = run_training(tv, dev, q, k, v, only, causal=causal, softcap=softcap, slopes=sl)
            assert int(dq[:, : first + 1].count_nonzero()) == 0 and int(dk.count_nonzero()) == 0
        _, dq, _, _ = run_training(tv, dev, q, k, v, go, causal=causal, softcap=softcap, slopes=sl)
        assert int(dq[:, : first + 1].count_nonzero()) == 0
