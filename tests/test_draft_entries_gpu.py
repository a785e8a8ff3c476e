"""GPU: probabilities that are none (negative, infinite, NaN) count as 0 wherever drafts are verified against them: in the
comparison, in what is left of the target's row, on either side."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ODD = (math.nan, -0.5, math.inf, -math.inf, -0.0)


def good(x):
    return x if 0.0 < x <= 3.402823466e38 else 0.0


def verify(p, q, draft, n, u):
    """One sequence, as defined; q None: certain drafts."""
    p = [[good(x) for x in row] for row in p]
    q = q if q is None else [[good(x) for x in row] for row in q]
    a = 0
    while a < n and u[a] * (1.0 if q is None else q[a][draft[a]]) < p[a][draft[a]]:
        a += 1
    row = p[a]
    if a < n:
        row = [0.0 if v == draft[a] else x for v, x in enumerate(row)] if q is None else [max(x - y, 0.0) for x, y in zip(row, q[a])]
        row = row if any(row) else p[a]
    target, sofar, token = u[-1] * math.fsum(row), 0.0, 0
    for v, x in enumerate(row):
        sofar += x
        if x > 0.0:
            token = v
            if sofar > target:
                break
    return a, draft[:a] + [token] + [-1] * (len(u) - 1 - a)


def check(gpu, p, q, draft, n, u):
    B, K1, V = p.shape
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    accepted, tokens = (torch.full(s, -9, dtype=torch.int32, device=DEV) for s in ((B,), (B, K1)))
    gpu.draft_verify(accepted, tokens, dev(p), dev(q), dev(draft), dev(n), dev(u), B, K1 - 1, V)
    gpu.synchronize()
    for b in range(B):
        a, t = verify(p[b].double().tolist(), None if q is None else q[b].double().tolist(), draft[b].tolist(),
                      K1 - 1 if n is None else int(n[b]), u[b].double().tolist())
        assert (int(accepted[b]), tokens[b].tolist()) == (a, t), b
    return accepted


def case(B, K, V, seed):
    g = torch.Generator().manual_seed(seed)
    rows = 2 * torch.randn(B, K + 1, V, generator=g)
    p = torch.softmax(rows, 2)
    q = torch.softmax(rows[:, :K] + 0.5 * torch.randn(B, K, V, generator=g), 2)
    draft = torch.multinomial(q.view(B * K, V), 1, generator=g).view(B, K).int()
    return p, q, draft, torch.rand(B, K + 1, generator=g)


@pytest.mark.parametrize("V,B", [(40, 16), (5000, 4), (20000, 4)])
@pytest.mark.parametrize("odd", ODD)
def test_entries_of_the_drafted_tokens(gpu, odd, V, B):
    """The entry that a draft is accepted by: of p, none is; of q, all are that the target has."""
    p, q, draft, u = case(B, 2, V, V)
    at = draft.long()[..., None]
    bad = p.clone()
    bad[:, :2] = p[:, :2].scatter(2, at, odd)
    assert (check(gpu, bad, q, draft, None, u) == 0).all()
    assert (check(gpu, bad, None, draft, None, u) == 0).all()
    assert (check(gpu, p, q.scatter(2, at, odd), draft, None, u) == 2).all()
    u[:, 0] = 0.0
    assert (check(gpu, bad, q, draft, None, u) == 0).all()


@pytest.mark.parametrize("V,B", [(40, 16), (5000, 4), (20000, 4)])
@pytest.mark.parametrize("odd", ODD)
def test_entries_of_the_other_tokens(gpu, odd, V, B):
    """A third of the drafts' entries, and some of the target's, are none; the first draft is refused: the token has p's own there."""
    p, q, draft, u = case(B, 2, V, V + 1)
    g = torch.Generator().manual_seed(7)
    hit_q, hit_p = torch.rand(q.shape, generator=g) < 1 / 3, torch.rand(p.shape, generator=g) < 0.1
    q[hit_q] = odd
    p[hit_p] = odd
    p[:, 0].scatter_(1, draft[:, :1].long(), 0.0)
    for x in (0.0, 0.3, 0.7, 0.999):
        u[:, 2] = x
        assert (check(gpu, p, q, draft, None, u) == 0).all()
    check(gpu, p, q, draft, torch.tensor([b % 3 for b in range(B)], dtype=torch.int32), u)
    p[:, :, 1:] = odd  # one token is left, of which the drafts' row takes all, or nothing
    p[:, :, 0], q[:, :, 0] = 0.25, 0.5
    draft[:] = 1
    check(gpu, p, q, draft, None, u)
