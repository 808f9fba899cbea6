"""Plain float64 evaluation of the attention operators on the CPU, with the error each rounding of the kernels may add.

Rounding to a type is off by at most u = finfo(type).eps / 2 relative to the value.  The kernels hold scores, maxima, sums and
states in float32 (unit 2^-24) and round: the softmax weights and the score gradients to the operands' 16-bit type in front of the
second products, the results once at the end.  `forward` / `backward` return values and element-wise bounds built from exactly that."""
import math

import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def sees(b, tq, tk, causal, prefix, documents, cache_len=None, count=None):
    """[b, tq, tk] truth values and [b, tq] places of the queries."""
    i, j = torch.arange(tq)[None, :, None], torch.arange(tk)[None, None, :]
    if cache_len is not None:
        place = cache_len[:, None] + torch.arange(tq)
        see = (j <= place[:, :, None]) | (j < prefix[:, None, None])
        return see & (j < (cache_len + count)[:, None, None]) & (i < count[:, None, None]), place
    place = (torch.arange(tq) + tk - tq)[None].expand(b, tq)
    see = torch.ones((b, tq, tk), dtype=torch.bool)
    if causal:
        see = (j <= place[:, :, None]) | (j < prefix[:, None, None])
    if documents is not None:
        see = see & (documents[:, :, None] == documents[:, None, :]) & (documents >= 0)[:, :, None]
    return see, place


def _clean(x, see_any):
    """Rows nobody sees hold whatever they hold: zero them for the float64 products."""
    return torch.where(see_any[..., None], x, torch.zeros((), dtype=x.dtype))


class Attention:
    """q [b, tq, hq, d], k, v [b, tk, hk, d] on the CPU in their own type; see [b, tq, tk]; place [b, tq]."""

    def __init__(self, q, k, v, see, place, scale=None, softcap=0.0, slopes=None):
        self.dtype, self.see = q.dtype, see
        b, tq, hq, d = q.shape
        tk, hk = k.shape[1], k.shape[2]
        self.shape, n = (b, tq, tk, hq, hk, d), hq // hk
        scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.scale = scale
        Q = _clean(q.double().transpose(1, 2), see.any(2)[:, None])
        K, V = (_clean(x.double().transpose(1, 2), see.any(1)[:, None]).repeat_interleave(n, 1) for x in (k, v))
        self.Q, self.K, self.V = Q, K, V
        s = Q @ K.transpose(2, 3) * scale
        size = Q.abs() @ K.abs().transpose(2, 3) * abs(scale)
        self.bend = torch.ones_like(s)
        if softcap > 0:
            th = torch.tanh(s / softcap)
            s, self.bend = softcap * th, 1 - th * th
        away = (place[:, :, None] - torch.arange(tk)).abs().double()[:, None]
        bias = slopes.double()[None, :, None, None] * away if slopes is not None else torch.zeros_like(s)
        s = s - bias
        m = see[:, None]
        s = torch.where(m, s, torch.full((), -math.inf, dtype=s.dtype))
        top = s.amax(-1, keepdim=True) if tk else torch.full((b, hq, tq, 1), -math.inf, dtype=s.dtype)
        w = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = w.sum(-1, keepdim=True)
        self.p = w / torch.where(total == 0, torch.ones_like(total), total)
        self.lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))[..., 0]
        self.out = self.p @ V
        # a score: d products and sums in float32, then cap and bias with a few more roundings (cap: a hardware exponential and
        # reciprocal, 2^-21 of the cap), log2(e) and the exponential's argument
        ds = F32 * ((d + 8) * size + 8 * (bias + 1) + 4 * torch.where(m, s, torch.zeros_like(s)).abs()) + (softcap * 2.0 ** -21 if softcap > 0 else 0)
        self.ds = torch.where(m, ds, torch.zeros_like(ds)).amax(-1, keepdim=True) if tk else torch.zeros((b, hq, tq, 1), dtype=s.dtype)
        u = unit(self.dtype) if self.dtype != torch.float32 else F32
        self.u = u
        # float16 holds multiples of 2^-24 below its smallest normal number 2^-14, so a rounding there is off by up to 2^-25 whatever the
        # value: weights (relative to a maximum of 1) and results alike
        self.step = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        W = self.p @ V.abs()
        seen = m.double() @ V.abs()
        self.out_tol = u * (W + self.out.abs()) * 1.01 + (2 * self.ds + (tk + 16) * F32) * W + self.step * seen + self.step + 1e-30

    def grads(self, go):
        b, tq, tk, hq, hk, d = self.shape
        n, u = hq // hk, self.u
        G = go.double().transpose(1, 2)
        G = torch.where(self.see.any(2)[:, None, :, None], G, torch.zeros_like(G))
        p, V, K, Q = self.p, self.V, self.K, self.Q
        dp = G @ V.transpose(2, 3)
        delta = (G * self.out).sum(-1, keepdim=True)
        core = p * (dp - delta) * self.bend
        ds = core * self.scale
        # errors of the score gradient: weights (2 ds + float32 sums), dp, delta (the rounded output), the cap's slope, its own rounding
        e_p = 2 * self.ds + (tk + 16) * F32
        e_dp = (d + 4) * F32 * (G.abs() @ V.abs().transpose(2, 3))
        e_delta = (G.abs() * (self.out_tol + u * self.out.abs())).sum(-1, keepdim=True) + (d + 4) * F32 * (G.abs() * self.out.abs()).sum(-1, keepdim=True)
        raw = p * (dp - delta).abs()
        e = (e_p + u * 1.01) * core.abs() + p * (e_dp + e_delta) + 2.0 ** -19 * raw + 8 * F32 * p * (dp.abs() + delta.abs())
        # float16 score gradients are rounded as multiples of 2^m: half the smallest step there is 2^-25 2^m.  m is a multiple of 8 with top / 2^m in
        # [2^-4, 2^4) for the largest output gradient top that the workgroup looks at, so 2^m <= 16 top <= 16 max |G|
        e = e + self.step * 16 * G.abs().amax() * self.see[:, None].double()
        e = e * abs(self.scale)
        dq = ds @ K
        dq_tol = e @ K.abs() + u * dq.abs() + self.step + (tk + 16) * F32 * (ds.abs() @ K.abs()) + 1e-30

        def shared(x):
            return x.view(b, hk, n, tk, d).sum(2)

        dk_h, dv_h = ds.transpose(2, 3) @ Q, p.transpose(2, 3) @ G
        dk, dv = shared(dk_h), shared(dv_h)
        terms = n * tq + 16
        dk_tol = shared(e.transpose(2, 3) @ Q.abs()) + u * dk.abs() + self.step + terms * F32 * shared(ds.abs().transpose(2, 3) @ Q.abs()) + 1e-30
        e_w = (u * 1.01 + 2 * self.ds + (tk + 16) * F32) * p + self.step * self.see[:, None].double()
        dv_tol = shared(e_w.transpose(2, 3) @ G.abs()) + u * dv.abs() + self.step + terms * F32 * shared(p.transpose(2, 3) @ G.abs()) + 1e-30
        rows = lambda x: x.transpose(1, 2)
        return [(rows(dq), rows(dq_tol)), (rows(dk), rows(dk_tol)), (rows(dv), rows(dv_tol))]

    def forward(self):
        return self.out.transpose(1, 2), self.out_tol.transpose(1, 2)


def within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite at {int((~torch.isfinite(got)).sum())} places"
    off = (got - want).abs() - tol
    if off.numel() and float(off.max()) > 0:
        at = int(off.argmax())
        raise AssertionError(f"{what}: {got.flatten()[at]:.8g} for {want.flatten()[at]:.8g}, off {float((got - want).abs().flatten()[at]):.3g}, bound {float(tol.flatten()[at]):.3g}, "
                             f"{int((off > 0).sum())} of {off.numel()} values")
