"""Attention in 64 bits, with the error that 32-bit sums may have, and the sequences of a test.

Error bounds (u = 2^-24, each rounding at most u relative). A score is a sum of HS products and a product with
the scale: off by at most e_s = (HS + 8) u scale sum |q k|; where an input is held as a sum of two shorter numbers
next to the largest of its row or tile, by HS 2^-38 scale max|q| max|k| more. p = exp(s - m) is then off by a factor
of e^(2 e_s) (its own score's error and the maximum's or the lse's), its exponent's rounding (|s - m| u) and the
exponential's 4 u; a sum of n such products adds n u. Every bound is the sum of the terms' sizes times these.
"""
import math

import torch

U = 2.0 ** -24


class Seqs:
    """Sequences with query lengths lq and key lengths lk; `gap` unused rows before each, `tail` behind the last."""

    def __init__(self, lq, lk=None, gap=0, tail=0):
        self.lq, self.lk = list(lq), list(lq if lk is None else lk)
        self.same = lk is None
        self.q, self.rows_q = self._place(self.lq, gap, tail)
        self.k, self.rows_k = (self.q, self.rows_q) if self.same else self._place(self.lk, gap, tail)

    @staticmethod
    def _place(lens, gap, tail):
        at, starts = 0, []
        for n in lens:
            starts.append(at + gap)
            at += gap + n
        return starts, at + tail


def allowed(nq, nk, causal, device="cpu"):
    i, j = torch.arange(nq, device=device)[:, None], torch.arange(nk, device=device)[None]
    return (j <= i + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool, device=device)


def _pieces(s, b, h, G, q, k, v):
    q0, k0, nq, nk = s.q[b], s.k[b], s.lq[b], s.lk[b]
    return (slice(q0, q0 + nq), slice(k0, k0 + nk), q[q0:q0 + nq, h].double(), k[k0:k0 + nk, h // G].double(),
            v[k0:k0 + nk, h // G].double())


def _score_error(q, k, scale, HS):
    big = q.abs().amax() * k.abs().amax() if q.numel() and k.numel() else 0.0
    return abs(scale) * ((HS + 8) * U * (q.abs() @ k.abs().T) + HS * 2.0 ** -38 * big)


def forward(s, q, k, v, scale, causal):
    """out, lse, and how far each may be off. Rows outside the sequences stay NaN."""
    NH, NKV, HS = q.shape[1], k.shape[1], q.shape[2]
    G = NH // NKV
    nan = lambda *a: torch.full(a, math.nan, dtype=torch.float64, device=q.device)  # noqa: E731
    out, lse, tol, tol_l = nan(*q.shape), nan(q.shape[0], NH), nan(*q.shape), nan(q.shape[0], NH)
    for b in range(len(s.lq)):
        for h in range(NH):
            rq, rk, x, y, z = _pieces(s, b, h, G, q, k, v)
            nq, nk = x.shape[0], y.shape[0]
            if not nq:
                continue
            ok = allowed(nq, nk, causal, q.device)
            S = (x @ y.T * scale).masked_fill(~ok, -math.inf)
            e = _score_error(x, y, scale, HS).masked_fill(~ok, 0.0)
            any_ = ok.any(1, keepdim=True)
            m = torch.where(any_, S.amax(1, keepdim=True) if nk else torch.zeros(nq, 1, dtype=S.dtype, device=S.device), 0.0)
            P = torch.exp(S - m)
            l = P.sum(1, keepdim=True)
            p = torch.where(any_, P / torch.where(any_, l, 1.0), 0.0)
            es = e.amax(1, keepdim=True) if nk else torch.zeros_like(m)
            depth = torch.where(ok, (m - S).clamp(0, 90), 0.0)
            rel = 2 * es + (depth + 4) * U
            out[rq, h] = p @ z
            terms = p * (2 * rel.amax(1, keepdim=True) if nk else rel) + p * (2 * nk + 16) * U
            size = z.abs()
            vmax = size.amax() if nk else 0.0
            tol[rq, h] = terms @ size + nk * 2.0 ** -38 * vmax * (p.amax(1, keepdim=True) if nk else 0.0)
            lse[rq, h] = (m + torch.log(l)).squeeze(1)
            tol_l[rq, h] = (es * 2 + (nk + 16) * U + 4 * U * (m.abs() + torch.log(l).abs().nan_to_num(0, 0, 0))).squeeze(1)
    return out, lse, tol, tol_l


def backward(s, q, k, v, out, lse, dout, scale, causal):
    """dq, dk, dv and how far each may be off, from the forward's (rounded) out and lse. Rows outside the sequences: 0."""
    NH, NKV, HS = q.shape[1], k.shape[1], q.shape[2]
    G = NH // NKV
    g = [torch.zeros(*t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    e = [torch.zeros_like(t) for t in g]
    for b in range(len(s.lq)):
        for h in range(NH):
            rq, rk, x, y, z = _pieces(s, b, h, G, q, k, v)
            nq, nk = x.shape[0], y.shape[0]
            if not nq or not nk:
                continue
            ok = allowed(nq, nk, causal, q.device)
            o, do = out[rq, h].double(), dout[rq, h].double()
            L = lse[rq, h, None].double()
            S = x @ y.T * scale
            P = torch.exp(S - L).masked_fill(~ok, 0.0)
            es = _score_error(x, y, scale, HS)
            D, Da = (do * o).sum(1, keepdim=True), (do.abs() * o.abs()).sum(1, keepdim=True)
            dP, dPa = do @ z.T, do.abs() @ z.abs().T
            # a product held as two shorter numbers, next to the largest of its tile
            floor = HS * 2.0 ** -38 * do.abs().amax() * z.abs().amax()
            dS = P * (dP - D) * scale
            rel = torch.where(ok, 2 * es + (S - L).abs().clamp(0, 90) * U + 8 * U, 0.0)
            size = P * (dPa + Da) * abs(scale)
            eS = size * (rel + (HS + 12) * U) + torch.where(ok, P * abs(scale) * floor, 0.0)
            bound = (HS * do.abs().amax() * z.abs().amax() + Da.amax()) * 2.0 ** -38 * abs(scale)  # of a held dS
            n = 2 * nq * G + 16
            g[0][rq, h] += dS @ y
            e[0][rq, h] += (eS + size * (2 * nk + 16) * U) @ y.abs() + bound * y.abs().sum(0) + \
                nk * 2.0 ** -38 * y.abs().amax() * size.amax()
            g[1][rk, h // G] += dS.T @ x
            e[1][rk, h // G] += (eS + size * n * U).T @ x.abs() + bound * x.abs().sum(0) + \
                nq * 2.0 ** -38 * x.abs().amax() * size.amax()
            g[2][rk, h // G] += P.T @ do
            e[2][rk, h // G] += (P * (rel + n * U)).T @ do.abs() + \
                nq * 2.0 ** -38 * do.abs().amax() * (P.amax() if P.numel() else 0.0) + 2.0 ** -38 * do.abs().sum(0)
    return g, e
