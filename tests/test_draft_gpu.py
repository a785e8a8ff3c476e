"""GPU: verification of drafted tokens against Python's floats, and a run of it with the cache in 8 bits."""
import math

import pytest
import torch

import cache8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(gpu, p, q, draft, n, u):
    """Tensors on the host; q and n may be None."""
    B, K1, V = p.shape
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    accepted, tokens = torch.full((B,), -9, dtype=torch.int32, device=DEV), torch.full((B, K1), -9, dtype=torch.int32, device=DEV)
    gpu.draft_verify(accepted, tokens, dev(p), dev(q), dev(draft), dev(n), dev(u), B, K1 - 1, V)
    rows = p.double().tolist(), None if q is None else q.double().tolist()
    for b in range(B):
        a, t = ref.verify(rows[0][b], None if q is None else rows[1][b], draft[b].tolist(), K1 - 1 if n is None else int(n[b]),
                          u[b].double().tolist())
        assert int(accepted[b]) == a and tokens[b].tolist() == t, b
    return accepted, tokens


def case(B, K, V, seed, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    rows = sharp * torch.randn(B, K + 1, V, generator=g)
    p = torch.softmax(rows, 2)
    q = torch.softmax(rows[:, :K] + 0.5 * torch.randn(B, K, V, generator=g), 2)
    draft = torch.multinomial(q.reshape(B * K, V), 1, generator=g).view(B, K).int() if K else torch.zeros(B, 0, dtype=torch.int32)
    n = torch.randint(0, K + 1, (B,), generator=g).int()
    return p, q, draft, n, torch.rand(B, K + 1, generator=g)


@pytest.mark.parametrize("V", [1, 2, 27, 63, 64, 65, 1000, 1023, 1025, 4099, 16385, 50257])
@pytest.mark.parametrize("K", [0, 1, 4, 8])
def test_verify(gpu, V, K):
    p, q, draft, n, u = case(3 if V > 5000 else 20, K, V, V + K)
    check(gpu, p, q, draft, n, u)
    check(gpu, p, None, draft, n, u)
    check(gpu, p, q, draft, None, u)
    gpu.synchronize()


def test_random_numbers_at_their_ends(gpu):
    """0 takes every draft that the target knows, and the first token; the largest below 1 the last that has any probability."""
    p, q, draft, n, u = case(8, 3, 500, 1)
    p[:, :, 400:] = 0.0
    p[:, :, :7] = 0.0
    for x in (0.0, 1.0 - 2.0 ** -24):
        u[:] = x
        accepted, tokens = check(gpu, p, q, draft, None, u)
        for b in range(8):
            a = int(accepted[b])
            assert 7 <= int(tokens[b, a]) < 400
            if x == 0.0 and a == 3:
                assert int(tokens[b, 3]) == 7
    u[:, 3] = 1.0  # no number of [0, 1): still a token
    check(gpu, p, q, draft, None, u)
    u[:] = math.nan
    accepted, _ = check(gpu, p, q, draft, None, u)
    assert (accepted == 0).all()
    gpu.synchronize()


def test_rows_that_agree_or_are_certain(gpu):
    p, q, draft, n, u = case(6, 2, 300, 2)
    q[:] = p[:, :2]
    u[:, 0] = 0.999
    check(gpu, p, q, draft, None, u)  # accepted always: u q < q
    u[:, 0] = 1.0  # refused by the number alone; nothing is left of p - q: the token is p's
    accepted, _ = check(gpu, p, q, draft, None, u)
    assert (accepted == 0).all()
    hot = torch.zeros_like(p)
    hot.scatter_(2, torch.randint(0, 300, (6, 3, 1)), 1.0)
    accepted, tokens = check(gpu, hot, None, hot[:, :2].argmax(2).int(), None, torch.rand(6, 3))
    assert (accepted == 2).all() and torch.equal(tokens.cpu().long(), hot.argmax(2))
    check(gpu, hot, None, (hot[:, :2].argmax(2).int() + 1) % 300, None, torch.rand(6, 3))
    gpu.synchronize()


def test_entries_that_are_no_probabilities_count_as_zero(gpu):
    p, q, draft, n, u = case(12, 2, 200, 3)
    p[:, :, 5], p[:, :, 6], p[:, :, 7], q[:, :, 8] = math.nan, -0.5, math.inf, math.nan
    draft.clamp_(min=9)
    check(gpu, p, q, draft, n, u)
    gpu.synchronize()


def test_borders_are_decided_exactly(gpu):
    """u q against p where single precision's product would round onto p."""
    V = 64
    p, q, u = torch.zeros(3, 2, V), torch.zeros(3, 1, V), torch.zeros(3, 2)
    u[:, 0] = 1.0 - 2.0 ** -24
    q[:, 0, 1] = 1.0 - 2.0 ** -23
    exact = float(u[0, 0].double() * q[0, 0, 1].double())  # between two floats
    low = torch.tensor(exact, dtype=torch.float32)
    for b, x in enumerate((low, torch.nextafter(low, torch.tensor(1.0)), torch.nextafter(low, torch.tensor(0.0)))):
        p[b, 0, 1] = x
    p[:, 0, 2] = p[:, 1, 3] = 0.25
    accepted, _ = check(gpu, p, q, torch.ones(3, 1, dtype=torch.int32), None, u)
    assert accepted.tolist() == [int(float(p[b, 0, 1]) > exact) for b in range(3)] and 0 < int(accepted.sum()) < 3


def test_what_is_reported(gpu):
    p, q, draft, n, u = case(4, 2, 50, 4)
    gpu.synchronize()
    for bad in (50, -1, 2 ** 31 - 1):
        d = draft.clone()
        d[1, 1] = bad
        u[1, 0] = 0.0
        check(gpu, p, q, d, None, u)
        with pytest.raises(gpu.UgkError, match="draft_verify"):
            gpu.synchronize()
    for bad in (3, -1):
        args = [t.to(DEV) for t in (p, q, draft)] + [torch.tensor([1, bad, 0, 2], dtype=torch.int32, device=DEV), u.to(DEV)]
        accepted, tokens = torch.empty(4, dtype=torch.int32, device=DEV), torch.empty(4, 3, dtype=torch.int32, device=DEV)
        gpu.draft_verify(accepted, tokens, *args, 4, 2, 50)
        with pytest.raises(gpu.UgkError, match="draft_verify"):
            gpu.synchronize()
        assert int(accepted[1]) <= max(0, min(bad, 2)) and (tokens[1] >= -1).all()
    p[2] = 0.0
    check(gpu, p, q, draft, None, u)  # token 0
    with pytest.raises(gpu.UgkError, match="without probabilities"):
        gpu.synchronize()
    gpu.synchronize()


def test_captured(gpu):
    p, q, draft, n, u = (t.to(DEV) for t in case(5, 4, 5000, 5))
    accepted, tokens = torch.empty(5, dtype=torch.int32, device=DEV), torch.empty(5, 5, dtype=torch.int32, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gpu.set_stream(s.cuda_stream)
        try:
            call = lambda: gpu.draft_verify(accepted, tokens, p, q, draft, n, u, 5, 4, 5000)  # noqa: E731
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call()
            for _ in range(3):
                u.uniform_()
                accepted.fill_(-9)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                got = accepted.tolist(), tokens.tolist()
                call()
                torch.cuda.synchronize()
                assert got == (accepted.tolist(), tokens.tolist())
        finally:
            s.synchronize()
            gpu.set_stream(None)


def test_generation_from_the_cache(gpu):
    """A small model's tokens from given random numbers: drafts verified against the cache in 8 bits, its blocks evicted where they
    got little weight, and the same done key by key in Python on what the cache holds."""
    NH, NKV, HS, V, nseq, K, cap, keep = 4, 2, 32, 27, 3, 3, 512, 4
    C = NH * HS
    g = torch.Generator(device=DEV)
    g.manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    emb, wqkv, head = rnd(V, C), rnd(C, (NH + 2 * NKV) * HS) / C ** 0.5, rnd(C, V) / C ** 0.5
    nb = cap // 64
    k8 = torch.zeros(nseq * nb, NKV, 64, HS, dtype=torch.int8, device=DEV)
    v8, ks = torch.zeros(nseq * nb, NKV, HS, 64, dtype=torch.int8, device=DEV), torch.zeros(nseq * nb, NKV, device=DEV)
    vs = torch.zeros_like(ks)
    table = torch.randperm(nseq * nb, generator=g, device=DEV).int().view(nseq, nb)
    lens = torch.zeros(nseq, dtype=torch.int32, device=DEV)
    weight, dropped = torch.zeros(nseq, nb, device=DEV), torch.zeros(nseq, dtype=torch.int32, device=DEV)
    models = [(ref.Model(NKV, HS), ref.Model(NKV, HS)) for _ in range(nseq)]

    def target(rows):
        """rows (nseq, n) of tokens, stored and attended to: logits (nseq, n, V)."""
        n = rows.shape[1]
        qkv = emb[rows.long()].view(nseq * n, C) @ wqkv
        lens.add_(n)
        ld = (NH + 2 * NKV) * HS
        a = gpu.Cache8(nseq=nseq, NH=NH, NKV=NKV, HS=HS, rows_q=nseq * n, max_q=n, max_k=cap, nblocks=nseq * nb, k_len=lens, table=table,
                       ldq=ld, ldk=ld, ldv=ld)
        flat, out = qkv.view(-1), torch.empty(nseq * n, C, device=DEV)
        gpu.cache8_store(k8, ks, v8, vs, flat[NH * HS:], flat[(NH + NKV) * HS:], a)
        few = n * (NH // NKV) <= 32
        gpu.cache8_attention(out, None, flat, k8, ks, v8, vs, a, weight=weight if few else None)
        t = qkv.view(nseq, n, NH + 2 * NKV, HS)
        for b in range(nseq):
            for m, x in zip(models[b], (t[b, :, NH:NH + NKV], t[b, :, NH + NKV:])):
                m.store(x, int(lens[b]))
            k, v = (m.values().to(DEV) for m in models[b])
            o, _, _, tol, _, _ = ref.attention(t[b, :, :NH], k, v, HS ** -0.5, True, few)
            assert ((out.view(nseq, n, NH, HS)[b].double() - o).abs() <= tol).all()
        return out.view(nseq, n, C) @ head

    rows = torch.randint(0, V, (nseq, 250), generator=g, device=DEV)
    last = target(rows)[:, -1].argmax(1).int()[:, None]
    gone = 0
    for step in range(40):
        q = torch.softmax(0.3 * rnd(nseq, K, V), 2)
        draft = torch.multinomial(q.view(-1, V), 1, generator=g).view(nseq, K).int()
        logits = target(torch.cat((last, draft), 1))
        p = torch.softmax(0.2 * logits, 2)
        u = torch.rand(nseq, K + 1, generator=g, device=DEV)
        accepted, tokens = torch.empty(nseq, dtype=torch.int32, device=DEV), torch.empty(nseq, K + 1, dtype=torch.int32, device=DEV)
        gpu.draft_verify(accepted, tokens, p, q, draft, None, u, nseq, K, V)
        for b in range(nseq):
            a, t = ref.verify(p[b].double().tolist(), q[b].double().tolist(), draft[b].tolist(), K, u[b].double().tolist())
            assert int(accepted[b]) == a and tokens[b].tolist() == t
        lens.sub_(K - accepted)  # the rows of drafts that were refused leave
        last = tokens.gather(1, accepted.long()[:, None])
        was = [(int(lens[b]), weight[b].tolist()) for b in range(nseq)]
        gpu.cache8_evict(table, lens, weight, dropped, table, lens, weight, nseq, nb, keep, 1, 2)
        for b in range(nseq):
            n, w = was[b]
            for m in models[b]:
                m.codes, m.scales = m.codes[:n], m.scales[:-(-n // 64)]
            if not int(dropped[b]):
                continue
            gone += 1
            order, _, _, d = ref.evict(list(range(nb)), n, w, keep, 1, 2)
            stay = order[:-(-n // 64) - d]
            for m in models[b]:
                m.codes = torch.cat([m.codes[64 * j:64 * j + 64] for j in stay])
                m.scales = [m.scales[j] for j in stay]
            assert len(models[b][0].codes) == int(lens[b])
    gpu.synchronize()
    assert gone > 0
