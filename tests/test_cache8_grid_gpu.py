"""GPU: many sequences of a table for very long ones: the launches go by the rows that there are and not by the longest that there could be."""
import pytest
import torch

import cache8_ref as ref
from test_cache8_gpu import DEV, gen, inside, ints, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nseq,some,HS,weigh", [(512, 512, 16, False), (512, 512, 16, True), (700, 700, 128, False), (4096, 11, 64, False)])
def test_many_sequences_of_a_long_table(gpu, nseq, some, HS, weigh):
    """One row of each of the first `some` sequences, 8 heads; blocks of the keys before are shared, the last is the sequence's own."""
    NKV, cap, common = 8, 131072, 64
    nb, HP, g = cap // 64, ref.padded(HS), gen(nseq)
    nblocks = common + some
    codes = lambda *s: torch.randint(-127, 128, s, dtype=torch.int8, generator=g, device=DEV)  # noqa: E731
    k8, v8 = codes(nblocks, NKV, 64, HP), codes(nblocks, NKV, HP, 64)
    k8[..., HS:], v8[:, :, HS:] = 0, 0
    ks, vs = (torch.exp2(torch.randint(-7, -4, (nblocks, NKV), generator=g, device=DEV).float()) for _ in "kv")
    long = {1: cap, 5: cap - 1, 10: 70001}
    keys = [long.get(b, 1 + b * 37 % 300) if b < some else 0 for b in range(nseq)]
    table = torch.randint(0, common, (nseq, nb), generator=g, device=DEV).int()
    for b in range(some):
        table[b, (keys[b] - 1) // 64] = common + b
    q, k, v = (rand(g, some, NKV, HS) for _ in "qkv")
    at = list(range(some)) + [some] * (nseq - some)
    a = gpu.Cache8(nseq=nseq, NH=NKV, NKV=NKV, HS=HS, rows_q=some, max_q=1, max_k=cap, nblocks=nblocks, q_start=ints(at),
                   q_end=ints([min(x + 1, some) for x in at]), k_len=ints(keys), table=table)
    out, lse = torch.full_like(q, 7.0), torch.full((some, NKV), 7.0, device=DEV)
    weight = torch.zeros(nseq, nb, device=DEV) if weigh else None
    kept = ks.clone(), vs.clone()
    gpu.cache8_store(k8, ks, v8, vs, k, v, a)
    back = torch.empty_like(k), torch.empty_like(v)
    gpu.cache8_load(*back, k8, ks, v8, vs, a)
    gpu.cache8_attention(out, lse, q, k8, ks, v8, vs, a, weight=weight)
    gpu.synchronize()
    assert torch.equal(ks[:common], kept[0][:common]) and torch.equal(vs[:common], kept[1][:common])
    uk, uv = ref.unpack(k8, ks, HS, False), ref.unpack(v8, vs, HS, True)
    for x, u, s in ((back[0], uk, ks), (back[1], uv, vs)):
        i = (torch.tensor(keys[:some], device=DEV) - 1) % 64
        held = u[common + torch.arange(some, device=DEV), :, i]
        assert torch.equal(x.double(), held)
    for x, y, s in ((back[0], k, ks), (back[1], v, vs)):  # half a step
        assert ((x.double() - y.double()).abs() <= 0.5 * s[common:].double()[..., None]).all()
    for b in sorted({0, 1, 2, 5, 7, 10, some // 2, some - 1} & set(range(some))):
        n = keys[b]
        o, l, w, tol, tol_l, tol_w = ref.attention(q[b:b + 1], ref.gather(uk, table[b], n), ref.gather(uv, table[b], n), HS ** -0.5, True, True)
        inside(out[b:b + 1], o, tol, f"out of {b}")
        inside(lse[b:b + 1], l, tol_l, f"lse of {b}")
        if weigh:
            inside(weight[b, :len(w)], w, tol_w + 2 * ref.U * w, f"weight of {b}")
            assert (weight[b, len(w):] == 0).all()
