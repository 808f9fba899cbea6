"""Tighter element-wise bounds than tests/attention_reference.py where float16 loses digits: the size of its subnormal numbers counts relative to what the kernels
scale by.

Score gradients: every column (a query of dq, a key of dk) is rounded where its largest score gradient so far is between 1 and 2^15, or brought there by a
power of two.  float16 holds multiples of 2^-24 at the lower end, so a rounding there is off by at most 2^-25 of the column's own largest one, whatever
other columns hold.

Softmax weights: in the forward pass the largest weight of a row is 2^7 or more when float16 rounds it, so a small one is off by 2^-32 of the largest; the
backward pass rounds 2^12 times the weight (at most 2^12), so by 2^-37.

Delta: for 16-bit operands the sum of p dp in float32; the rounded output's part in it is corrected.

Caps: 16-bit operands take a short tanh that is off by 2^-21 up to a cap of 64; beyond, and for float32, the error is relative: the quotient by the cap, the
tanh (its own form and one hardware exponential and reciprocal) and the product with the cap are within 2^-20 of the capped score together."""
import torch

import attention_reference as R


class Tight(R.Attention):
    def __init__(self, q, k, v, see, place, scale=None, softcap=0.0, slopes=None):
        super().__init__(q, k, v, see, place, scale, softcap, slopes)
        b, tq, tk, hq, hk, d = self.shape
        F32, m, half = R.F32, see[:, None], self.dtype == torch.float16
        if softcap > (64.0 if self.dtype != torch.float32 else 0.0):
            # the reference's score error with this one in place of 2^-21 of the cap (not by a difference: a cap of 1e38 leaves nothing beside it)
            size = self.Q.abs() @ self.K.abs().transpose(2, 3) * abs(self.scale)
            capped = softcap * torch.tanh(self.Q @ self.K.transpose(2, 3) * self.scale / softcap)
            bias = slopes.double()[None, :, None, None] * (place[:, :, None] - torch.arange(tk)).abs().double()[:, None] if slopes is not None else torch.zeros_like(capped)
            ds = F32 * ((d + 8) * size + 8 * (bias + 1) + 4 * (capped - bias).abs()) + 2.0 ** -20 * capped.abs()
            self.ds = torch.where(m, ds, torch.zeros_like(ds)).amax(-1, keepdim=True)
        W = self.p @ self.V.abs()
        self.out_tol = self.u * (W + self.out.abs()) * 1.01 + (2 * self.ds + (tk + 16) * F32) * W + 1e-30
        if half:
            self.out_tol = self.out_tol + 2.0 ** -32 * (m.double() @ self.V.abs()) + 2.0 ** -25

    def grads(self, go):
        b, tq, tk, hq, hk, d = self.shape
        n, u, F32 = hq // hk, self.u, R.F32
        G = go.double().transpose(1, 2)
        G = torch.where(self.see.any(2)[:, None, :, None], G, torch.zeros_like(G))
        p, V, K, Q, see = self.p, self.V, self.K, self.Q, self.see[:, None].double()
        half = self.dtype == torch.float16
        dp = G @ V.transpose(2, 3)
        delta = (G * self.out).sum(-1, keepdim=True)
        core = p * (dp - delta) * self.bend
        # the same roundings as in the reference: weights, dp, delta (of the rounded output), the cap's slope, the score gradient's own
        e_p = 2 * self.ds + (tk + 16) * F32
        e_dp = (d + 4) * F32 * (G.abs() @ V.abs().transpose(2, 3))
        e_delta = (G.abs() * (self.out_tol + u * self.out.abs())).sum(-1, keepdim=True) + (d + 4) * F32 * (G.abs() * self.out.abs()).sum(-1, keepdim=True)
        off = e_delta
        if self.dtype != torch.float32:
            # the sum of p dp itself, in float32
            e_delta = ((e_p + (tk + 16) * F32) * p * dp.abs() + p * e_dp).sum(-1, keepdim=True) + 8 * F32 * (delta.abs() + off)
        e = (e_p + u * 1.01) * core.abs() + p * (e_dp + e_delta) + 2.0 ** -19 * p * (dp - delta).abs() + 8 * F32 * p * (dp.abs() + delta.abs())
        size = core.abs() + e
        step = 2.0 ** -25 if half else 0.0
        group = lambda x: x.view(b, hk, n, tq, tk)
        e_q = (e + step * size.amax(-1, keepdim=True) * see) * abs(self.scale)
        e_k = (e + step * group(size).amax((2, 3), keepdim=True).expand(b, hk, n, 1, tk).reshape(b, hq, 1, tk) * see) * abs(self.scale)
        least = 2.0 ** -25 if half else 0.0             # of the results
        ds = core * self.scale
        shared = lambda x: x.view(b, hk, n, tk, d).sum(2)
        dq, dk, dv = ds @ K, shared(ds.transpose(2, 3) @ Q), shared(p.transpose(2, 3) @ G)
        # the correction of dq: what delta of the rounded output is off, times a mean of keys whose weights are rounded
        mean = off * ((u * 1.01 * p + least * see) @ K.abs()) * abs(self.scale) if self.dtype != torch.float32 else 0.0
        dq_tol = e_q @ K.abs() + mean + u * dq.abs() + least + (tk + 16) * F32 * (ds.abs() @ K.abs()) + 1e-30
        terms = n * tq + 16
        dk_tol = shared(e_k.transpose(2, 3) @ Q.abs()) + u * dk.abs() + least + terms * F32 * shared(ds.abs().transpose(2, 3) @ Q.abs()) + 1e-30
        e_w = (u * 1.01 + e_p) * p + (2.0 ** -37 * see if half else 0.0)
        dv_tol = shared(e_w.transpose(2, 3) @ G.abs()) + u * dv.abs() + least + terms * F32 * shared(p.transpose(2, 3) @ G.abs()) + 1e-30
        rows = lambda x: x.transpose(1, 2)
        return [(rows(dq), rows(dq_tol)), (rows(dk), rows(dk_tol)), (rows(dv), rows(dv_tol))]
