"""GPU: the new operators in a run, as a network calls them: a block's training pass (attention, residual dropout, LayerNorm
and their gradients), and generation (a prompt, then single tokens against the cache that both wrote)."""
import pytest
import torch

import att_ref
import drop_ref
from att_ref import Seqs

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
P, SEED = 0.1, 77


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"{what}: worst {float((err / tol.clamp(min=1e-300)).max()):.3g} of the bound"


def layernorm64(x, w, b):
    mean = x.mean(1, keepdim=True)
    r = ((x - mean) ** 2).mean(1, keepdim=True).add(1e-5).rsqrt()
    return (x - mean) * r * w + b, (x - mean) * r, r


@pytest.mark.parametrize("T,NH,HS", [(70, 3, 64), (9, 2, 33), (130, 2, 128)])
def test_training_pass_of_a_block(gpu, T, NH, HS):
    """qkv -> attention -> res = x + dropout(attention) -> LayerNorm, and back to dqkv and dx. Each step is held to 64
    bits of the step's own inputs in this run."""
    B, C = 2, NH * HS
    rows, n = B * T, B * T * C
    g = torch.Generator(device=DEV)
    g.manual_seed(T)
    qkv, x, dout = rand(g, rows, 3 * C), rand(g, rows, C), rand(g, rows, C)
    w, b = rand(g, C, scale=0.1) + 1.0, rand(g, C, scale=0.1)
    flat = qkv.view(-1)
    a = gpu.Attention(B, NH, NH, HS, rows, rows, T, T, ldq=3 * C, ldk=3 * C, ldv=3 * C)
    e = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    att, lse, res, out, mean, rstd = e(rows, C), e(rows, NH), e(rows, C), e(rows, C), e(rows), e(rows)
    gpu.attention_forward(att, lse, flat, flat[C:], flat[2 * C:], a)
    gpu.dropout_residual_layernorm_forward(res, out, mean, rstd, x, att, w, b, B, T, C, P, SEED, 3, 1)
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    dres, dw, db, dx, datt, dqkv = z(rows, C), z(C), z(C), z(rows, C), z(rows, C), z(rows, 3 * C)
    gpu.layernorm_dropout_residual_backward(dres, dw, db, dx, datt, dout, res, w, mean, rstd, B, T, C, P, SEED, 3, 1)
    df = dqkv.view(-1)
    gpu.attention_backward(df, df[C:], df[2 * C:], datt, flat, flat[C:], flat[2 * C:], att, lse, a)
    gpu.synchronize()

    s = Seqs([T] * B)
    heads = lambda t, i: t[:, i * C:(i + 1) * C].unflatten(1, (NH, HS))  # noqa: E731
    q, k, v = (heads(qkv, i) for i in range(3))
    want, wl, tol, tol_l = att_ref.forward(s, q, k, v, HS ** -0.5, True)
    close(att.view(rows, NH, HS), want, tol, "attention")
    close(lse, wl, tol_l, "lse")
    kept = drop_ref.keep(n, P, SEED, 3, 1)
    drop = lambda t: torch.from_numpy(drop_ref.drop(t.cpu().numpy().reshape(-1), kept, P)).view(rows, C).to(DEV)  # noqa: E731
    assert torch.equal(res, x + drop(att))
    y, h, r = layernorm64(res.double(), w.double(), b.double())
    # the mean and the sum of squares each add C terms (C U), then a subtraction, two products and a sum
    spread = res.double().abs().amax(1, keepdim=True) * r + h.abs()
    close(out, y, (2 * C + 16) * U * spread * w.abs() + 2 * U * b.abs(), "LayerNorm")
    gw = dout.double() * w.double()
    m1, m2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    size = (gw.abs() + gw.abs().mean(1, keepdim=True) + h.abs() * (gw.abs() * (h.abs() + spread)).mean(1, keepdim=True)
            + spread * m2.abs()) * r
    close(dres, (gw - m1 - h * m2) * r, (4 * C + 32) * U * size, "dres")
    assert torch.equal(dx, dres) and torch.equal(datt, drop(dres))
    got = [heads(dqkv, i) for i in range(3)]
    want, tol = att_ref.backward(s, q, k, v, att.view(rows, NH, HS), lse, datt.view(rows, NH, HS), HS ** -0.5, True)
    for name, u, t, bound in zip(("dq", "dk", "dv"), got, want, tol):
        close(u, t, bound, name)


@pytest.mark.parametrize("NH,NKV,HS,lens,more", [(4, 4, 64, [5, 90, 1], 40), (8, 2, 128, [130, 33], 30), (3, 1, 40, [0, 7], 66)])
def test_generation_from_a_cache(gpu, NH, NKV, HS, lens, more):
    """Prompts of different lengths, then one token of each sequence at a time against the filled part of its cache, as one
    pass over the whole sequences gives. The rest of the cache holds NaN."""
    nseq, cap = len(lens), max(lens) + more + 3
    g = torch.Generator(device=DEV)
    g.manual_seed(HS)
    total = [m + more for m in lens]
    q = [rand(g, t, NH * HS) for t in total]
    k, v = ([rand(g, t, NKV * HS) for t in total] for _ in range(2))
    ck, cv = (torch.full((nseq * cap, NKV * HS), float("nan"), device=DEV) for _ in range(2))
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device=DEV)  # noqa: E731
    start = [i * cap for i in range(nseq)]
    got = [torch.empty(t, NH * HS, device=DEV) for t in total]

    def step(first, count, max_q):
        rows = sum(count)
        cu = [sum(count[:i]) for i in range(nseq + 1)]
        for i in range(nseq):
            for c, t in ((ck, k), (cv, v)):
                c[start[i] + first[i]:start[i] + first[i] + count[i]] = t[i][first[i]:first[i] + count[i]]
        qs = torch.cat([q[i][first[i]:first[i] + count[i]] for i in range(nseq)])
        out = torch.empty_like(qs)
        a = gpu.Attention(nseq, NH, NKV, HS, rows, nseq * cap, max_q, cap, q_start=ints(cu[:-1]), q_end=ints(cu[1:]),
                          k_start=ints(start), k_end=ints([start[i] + first[i] + count[i] for i in range(nseq)]))
        gpu.attention_forward(out, None, qs, ck, cv, a)
        for i in range(nseq):
            got[i][first[i]:first[i] + count[i]] = out[cu[i]:cu[i + 1]]

    step([0] * nseq, lens, max(lens))
    for t in range(more):
        step([m + t for m in lens], [1] * nseq, 1)
    gpu.synchronize()
    s = Seqs(total)
    cat = lambda t, h: torch.cat(t).unflatten(1, (h, HS))  # noqa: E731
    want, _, tol, _ = att_ref.forward(s, cat(q, NH), cat(k, NKV), cat(v, NKV), HS ** -0.5, True)
    close(cat(got, NH), want, tol, "out")
