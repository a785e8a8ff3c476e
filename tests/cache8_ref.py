"""A cache in 8 bits in plain Python and 64 bits: what it holds after stores, attention over it with the error that it may
have, eviction, and the verification of drafts.

Error bounds of the attention (u = 2^-24). A row of q is off by 2^-30 of its largest element (whole numbers of 31 bits), or by
2^-23 of each and 2^-38 of the largest (two halves). A score is then a sum of HS products, exact in the first case and of 2 HS
roundings in the second, and up to 8 roundings of the parts' sum and the factor: off by e_s = ((2 HS + 8) u + 2^-23) scale sum |q k|
+ 2^-30 scale max|q| sum |k| at most. p = 2^(s - m) is off by a factor of e^(2 e_s) (its own score's error and the
maximum's), the rounding of its exponent (|s - m| u, and as much for the block's maximum against the row's) and of three exponentials (4 u each).
A weight is held to 2^-31 of the block's largest, or 2^-23 of itself and 2^-38 of that (of two halves, as seen through the
values' scales: of the largest contribution), and a block's largest is at most the row's. A sum of n
products adds n u (2 n for two halves), the blocks' and parts' factors 16 u.
"""
import math

import torch

U = 2.0 ** -24
BLOCK = 64


def padded(HS):
    return (HS + 15) // 16 * 16


def place():
    i = torch.arange(BLOCK)
    return i % 16 * 4 + i // 16


def scale_for(top):
    """The least power of two s, 2^-126 to 2^121, with top <= 127 s."""
    if top == 0:
        return 0.0
    e = -126
    while e < 121 and top > 127 * math.ldexp(1.0, e):
        e += 1
    return math.ldexp(1.0, e)


def unpack(code, scale, HS, values):
    """(blocks, NKV, 64, HS) in 64 bits, of device buffers (blocks, NKV, ...)."""
    t = code[..., place().to(code.device)].transpose(2, 3) if values else code
    return t[..., :HS].double() * scale.double()[:, :, None, None]


def gather(block, table, n):
    """Keys [0, n) of a sequence whose blocks `table` lists: (n, NKV, HS)."""
    t = block[table.long()]
    return t.permute(0, 2, 1, 3).reshape(-1, t.shape[1], t.shape[3])[:n]


class Model:
    """One sequence's keys (or values) as stores leave them: a list of codes and the scale per block and head."""

    def __init__(self, NKV, HS):
        self.codes, self.scales = torch.zeros(0, NKV, HS, dtype=torch.float64), []

    def store(self, rows, end):
        """rows (n, NKV, HS) as the last of `end` keys."""
        rows = rows.double().cpu()
        begin = end - len(rows)
        self.codes = torch.cat((self.codes[:begin], torch.zeros_like(rows)))
        for j in range(begin // BLOCK, (end + BLOCK - 1) // BLOCK):
            lo, mid, hi = j * BLOCK, max(begin, j * BLOCK), min(end, (j + 1) * BLOCK)
            new = rows[mid - begin:hi - begin]
            s = torch.tensor([scale_for(float(x)) for x in new.abs().amax((0, 2))], dtype=torch.float64)
            del self.scales[j + 1:]
            if mid > lo:
                was = self.scales[j]
                s = torch.maximum(s, was)
                f = torch.where(s > 0, was / torch.where(s > 0, s, 1.0), 1.0)
                self.codes[lo:mid] = (self.codes[lo:mid] * f[:, None]).round()
                self.scales[j] = s
            else:
                del self.scales[j:]
                self.scales.append(s)
            self.codes[mid:hi] = (new / torch.where(s > 0, s, 1.0)[:, None]).round().clamp(-127, 127)

    def values(self):
        return torch.cat([self.codes[j * BLOCK:(j + 1) * BLOCK] * s[:, None] for j, s in enumerate(self.scales)] or [self.codes])


def attention(q, k, v, scale, causal, few):
    """One sequence: q (n, NH, HS), k and v (m, NKV, HS) in 64 bits. out, lse, the blocks' weights, and how far each may be off."""
    n, NH, HS = q.shape
    m, NKV = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    blocks = (m + BLOCK - 1) // BLOCK
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((n, NH), -math.inf, dtype=torch.float64, device=q.device)
    tol_l = torch.zeros_like(lse)
    weight = torch.zeros(blocks, dtype=torch.float64, device=q.device)
    tol_w = torch.zeros_like(weight)
    if not m:
        return out, lse, weight, tol, tol_l, tol_w
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None]
    ok = (j <= i + m - n) if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
    any_ = ok.any(1, keepdim=True)
    for h in range(NH):
        x, y, z = q[:, h], k[:, h // (NH // NKV)], v[:, h // (NH // NKV)]
        S = (x @ y.T * scale).masked_fill(~ok, -math.inf)
        e = abs(scale) * (((2 * HS + 8) * U + 2.0 ** -23) * (x.abs() @ y.abs().T) +
                          2.0 ** -30 * x.abs().amax(1, keepdim=True) * y.abs().sum(1)[None])
        es = e.masked_fill(~ok, 0.0).amax(1, keepdim=True)
        top = torch.where(any_, S.amax(1, keepdim=True), 0.0)
        P = torch.exp(S - top)
        l = P.sum(1, keepdim=True)
        p = torch.where(any_, P / torch.where(any_, l, 1.0), 0.0)
        depth = torch.where(ok, (top - S).clamp(0, 100), 0.0)
        rel = 2 * es + (3 * depth / math.log(2.0) + 16) * U
        terms = p * (2 * rel + (2 * m + 32) * U + 2.0 ** -23)
        held = 2.0 ** (-31 if few else -38) * torch.where(any_, 1.0 / torch.where(any_, l, 1.0), 0.0)  # of the largest weight
        out[:, h] = p @ z
        tol[:, h] = terms @ z.abs() + 2 * held * z.abs().sum(0) + 2 * U * out[:, h].abs()
        lse[:, h] = (top + torch.log(l)).squeeze(1)
        tol_l[:, h] = (2 * es + (m + 32) * U + 4 * U * (top.abs() + torch.log(l).abs())).squeeze(1)
        pad = lambda t: torch.nn.functional.pad(t.sum(0), (0, blocks * BLOCK - m)).view(blocks, BLOCK).sum(1)  # noqa: E731
        weight += pad(p)
        tol_w += pad(terms * 2) + pad(p) * (n * NH + 64) * U
    return out, lse, weight, tol, tol_l, tol_w


def evict(table, length, weight, keep, first, recent):
    """One sequence: (row of the table, length, weights, blocks gone). Lists."""
    n = -(-length // BLOCK)
    d = max(0, n - keep)
    key = lambda i: (1, 0.0, i) if weight[i] != weight[i] else (0, weight[i], i)  # noqa: E731
    gone = set(sorted(range(first, n - recent), key=key)[:d])
    stay = [i for i in range(n) if i not in gone]
    order = stay + list(range(n, len(table))) + sorted(gone)
    return [table[i] for i in order], length - BLOCK * d, [weight[i] for i in stay] + [0.0] * (len(table) - len(stay)), d


def verify(p, q, draft, n, u):
    """One sequence in Python's floats: (accepted, tokens). p, q: lists of rows of floats; q None: certain drafts."""
    K, a = len(p) - 1, 0
    while a < n and 0 <= draft[a] < len(p[a]) and u[a] * (1.0 if q is None else q[a][draft[a]]) < p[a][draft[a]]:
        a += 1
    good = lambda x: x if 0.0 < x <= 3.402823466e38 else 0.0  # noqa: E731
    whole = [good(x) for x in p[a]]
    row = whole
    if a < n:
        row = [0.0 if v == draft[a] else x for v, x in enumerate(whole)] if q is None else [good(x - y) for x, y in zip(p[a], q[a])]
        if not any(row):
            row = whole
    target, sofar, token = u[K] * math.fsum(row), 0.0, 0
    for v, x in enumerate(row):
        sofar += x
        if x > 0.0:
            token = v
            if sofar > target:
                break
    return a, list(draft[:a]) + [token] + [-1] * (K - a)
