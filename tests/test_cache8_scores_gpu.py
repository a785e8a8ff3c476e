"""GPU: attention over the cache in 8 bits for scores far beyond 2^20, which a row's weights have to survive: one key has all of the
weight, or equal scores share it.

What is known there without an exponential: a row's result lies between the least and the largest of the values that it sees; where the
best score is ahead of the others by more than the scores' errors (e_s each, as cache8_ref derives it) and 200, its key has the weight 1
and the others, below e^-200, none (weights are held to 2^-38 at the best, sums to 2^-24); and keys that are the same have the same score, bit by bit.
"""
import math

import pytest
import torch

import cache8_ref as ref
from test_cache8_gpu import DEV, attend, filled, inside, place_rows, rand

pytestmark = pytest.mark.gpu
U = ref.U


def scores(q, k, scale, causal):
    """(rows, heads, keys) in 64 bits, -infinity where masked, and the error of each."""
    n, NH, HS = q.shape
    m, NKV = k.shape[:2]
    q, k = q.double(), k.double().repeat_interleave(NH // NKV, 1)
    S = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()).transpose(0, 1) * scale
    e = abs(scale) * (((2 * HS + 8) * U + 2.0 ** -23) * torch.matmul(q.abs().transpose(0, 1), k.abs().permute(1, 2, 0).contiguous()).transpose(0, 1) +
                      2.0 ** -30 * q.abs().amax(2, keepdim=True) * k.abs().sum(2).T[None])
    i, j = torch.arange(n, device=DEV)[:, None, None], torch.arange(m, device=DEV)
    ok = (j <= i + m - n) if causal else torch.ones(n, 1, m, dtype=torch.bool, device=DEV)
    return S.masked_fill(~ok, -math.inf), e, ok.expand_as(S)


def look(c, q, out, L, weight, starts, lens, keys, scale, causal):
    """The checks of the module's first lines; the share of rows whose best score is clear."""
    clear_rows = []
    for b, n in enumerate(lens):
        at, m = slice(starts[b], starts[b] + n), keys[b]
        NH, NKV = q.shape[1], c.NKV
        v = c.values(b, m, "v").repeat_interleave(NH // NKV, 1)  # (m, NH, HS)
        S, e, ok = scores(q[at], c.values(b, m, "k"), scale, causal)
        top, best = S.max(2)
        es = e.masked_fill(~ok, 0.0).amax(2)
        second = S.scatter(2, best[..., None], -math.inf).amax(2)
        clear = top - second > 2 * es + 200
        clear_rows.append(clear.double().mean().item())
        most = v.abs().amax(0)[None]
        o, last = out[at].double(), ok[:, 0].sum(1) - 1  # a row sees the keys up to its last
        slack = (2 * m + 64) * U * most + 2.0 ** -30 * m * most
        assert (o >= v.cummin(0).values[last] - slack).all() and (o <= v.cummax(0).values[last] + slack).all(), b
        want = v[best, torch.arange(NH, device=DEV)]  # (n, NH, HS)
        err = ((o - want).abs() <= 16 * U * want.abs()) | ~clear[..., None]
        assert err.all(), (b, int((~err).sum()))
        # lse: the sum is between 1 and m
        l = L[at].double()
        assert l.isfinite().all()
        tol = 2 * es + 8 * U * top.abs() + math.log(m) + 1.0
        assert ((l - top).abs() <= tol).all(), b
        assert ((l - top).abs() <= 2 * es + 8 * U * top.abs())[clear].all(), b
        if weight is not None:
            got = weight[b].double()
            total = float(n * NH)
            assert abs(float(got.sum()) - total) <= total * (2 * m + n * NH + 128) * U
            if clear.all():
                count = torch.zeros_like(got).index_add_(0, (best // 64).flatten(), torch.ones(n * NH, dtype=torch.float64, device=DEV))
                assert ((got - count).abs() <= (16 + n * NH) * U * count).all(), b
    return sum(clear_rows) / len(clear_rows)


@pytest.mark.parametrize("HS", [64, 128])
@pytest.mark.parametrize("cap", [200, 5000])
@pytest.mark.parametrize("lq", [1, 5, 20, 40, 100])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_beyond_what_a_float_has_behind_the_point(gpu, sign, lq, cap, HS):
    """Scores of 2^20 to 2^120; negative: all of them, so that the best is the least far below zero."""
    NH, NKV = 2, 2
    keys, lens = [cap - 70, cap], [lq, (lq + 1) // 2]
    c, g = filled(gpu, 2, cap, NKV, HS, keys, size=lambda k, v: k.abs_() if sign < 0 else None)
    starts, rows = place_rows(lens)
    base = rand(g, rows, NH, HS)
    if sign < 0:
        base = -base.abs()
    for power in (20, 22, 25, 28, 33, 41, 64, 90, 118):
        q = base * 2.0 ** power
        for causal in (True, False):
            for weigh in (False, True):
                w = torch.zeros(c.table.shape, device=DEV) if weigh else None
                out, L = attend(gpu, c, NH, q, starts, lens, keys, rows, causal, w)
                gpu.synchronize()
                share = look(c, q, out, L, w, starts, lens, keys, HS ** -0.5, causal)
                assert share > 0.8 or power < 22, (power, causal, share)


@pytest.mark.parametrize("spread", [0, 60])
@pytest.mark.parametrize("cap", [64, 200, 5000])
@pytest.mark.parametrize("lq", [1, 5, 20, 40, 100])
def test_equal_scores_of_any_size_share_the_weight(gpu, lq, cap, spread):
    """All keys of a head are one: a row's result is the mean of the values, whatever the score and the scales of the blocks' values."""
    NH, NKV, HS = 4, 2, 64

    def size(k, v):
        k[:] = k[:1]
        v *= torch.exp2(spread * (torch.arange(len(v), device=DEV) // 64 % 3 - 1.0))[:, None, None]
    c, g = filled(gpu, 1, cap, NKV, HS, [cap], size=size)
    base = rand(g, lq, NH, HS)
    k, v = (c.values(0, cap, n).repeat_interleave(2, 1) for n in "kv")
    assert (k == k[:1]).all()
    for power in (10, 22, 26, 30, 34, 41, 64, 90, 118):
        q = base * 2.0 ** power
        for weigh in (False, True):
            w = torch.zeros(c.table.shape, device=DEV) if weigh else None
            out, L = attend(gpu, c, NH, q, [0], [lq], [cap], lq, False, w)
            gpu.synchronize()
            # a sum of cap products and its quotient; weights of 31 bits, or of two halves
            tol = (2 * cap + 64) * U * v.abs().mean(0) + 2.0 ** -30 * v.abs().sum(0) / cap
            inside(out, v.mean(0)[None].expand(lq, NH, HS), tol[None].expand(lq, NH, HS), f"out at 2^{power}")
            S, e, _ = scores(q, c.values(0, cap, "k"), HS ** -0.5, False)
            inside(L, S[..., 0] + math.log(cap), 2 * e[..., 0] + 8 * U * S[..., 0].abs() + (cap + 64) * U, f"lse at 2^{power}")
            if weigh:
                n = torch.full((cap // 64 + (cap % 64 > 0),), 64.0, dtype=torch.float64, device=DEV)
                n[-1] = cap - 64 * (len(n) - 1)
                inside(w[0], n / cap * lq * 2 * NKV, n / cap * lq * 2 * NKV * (2 * cap + lq * NH + 128) * U, f"weight at 2^{power}")


@pytest.mark.parametrize("lq", [1, 5, 20, 40, 100])
def test_a_far_score_in_one_row_leaves_the_others_alone(gpu, lq):
    """Rows of one call, some with scores beyond 2^20: the others' bits are those of the call without them."""
    NH, NKV, HS, cap = 2, 2, 64, 700
    c, g = filled(gpu, 1, cap, NKV, HS, [cap])
    q = rand(g, lq, NH, HS)
    want, L0 = attend(gpu, c, NH, q, [0], [lq], [cap], lq)
    far = q.clone()
    far[::3, 0] *= 2.0 ** 40
    got, L = attend(gpu, c, NH, far, [0], [lq], [cap], lq)
    gpu.synchronize()
    same = torch.ones(lq, NH, dtype=torch.bool, device=DEV)
    same[::3, 0] = False
    assert torch.equal(got[same], want[same]) and torch.equal(L[same], L0[same])
    look(c, far, got, L, None, [0], [lq], [cap], HS ** -0.5, True)
