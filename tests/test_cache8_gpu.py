"""GPU: the cache in 8 bits against its plain form and 64 bits: stores whole and piece by piece, attention at the lengths, heads,
strides and masks where it can go wrong, the blocks' weights, eviction, reports of bad arguments, graphs, streams."""
import math

import pytest
import torch

import cache8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Cache:
    """A cache of nseq sequences of up to `cap` keys, its blocks dealt out in a random order among `spare` others, every byte filled
    beforehand."""

    def __init__(self, gpu, nseq, cap, NKV, HS, seed=1, spare=3, ld=None):
        self.gpu, self.nseq, self.cap, self.NKV, self.HS = gpu, nseq, cap, NKV, HS
        nb = ld or (cap + 63) // 64
        self.nblocks = nseq * nb + spare
        g, HP = gen(seed), ref.padded(HS)
        assert gpu.cache8_bytes(self.nblocks, NKV, HS) == self.nblocks * NKV * 64 * HP
        fill = lambda *s: torch.randint(-128, 128, s, dtype=torch.int8, generator=g, device=DEV)  # noqa: E731
        self.k8, self.v8 = fill(self.nblocks, NKV, 64, HP), fill(self.nblocks, NKV, HP, 64)
        self.ks, self.vs = torch.full((self.nblocks, NKV), 0.5, device=DEV), torch.full((self.nblocks, NKV), 0.25, device=DEV)
        self.table = torch.randperm(self.nblocks, generator=g, device=DEV)[:nseq * nb].int().view(nseq, nb)

    def parts(self):
        return self.k8, self.ks, self.v8, self.vs

    def call(self, NH, starts, lens, keys, rows=None, **kw):
        rows = max([a + n for a, n in zip(starts, lens)], default=0) if rows is None else rows
        base = dict(nseq=self.nseq, NH=NH, NKV=self.NKV, HS=self.HS, rows_q=rows, max_q=max(lens, default=0), max_k=self.cap,
                    nblocks=self.nblocks, q_start=ints(starts), q_end=ints([a + n for a, n in zip(starts, lens)]), k_len=ints(keys),
                    table=self.table)
        base.update(kw)
        return self.gpu.Cache8(**base)

    def values(self, b, n, name):
        code, scale = (self.k8, self.ks) if name == "k" else (self.v8, self.vs)
        return ref.gather(ref.unpack(code, scale, self.HS, name == "v"), self.table[b], n)


def place_rows(lens, gap=1, tail=2):
    at, starts = 0, []
    for n in lens:
        starts.append(at + gap)
        at += gap + n
    return starts, at + tail


def view(buf, rows, heads, HS, ld):
    return buf.as_strided((rows, heads, HS), (ld, HS, 1), buf.storage_offset())


HEADS = [(1, 64), (2, 128), (3, 16), (2, 50), (1, 33), (2, 1), (2, 80), (1, 112), (2, 96)]


@pytest.mark.parametrize("NKV,HS", HEADS)
@pytest.mark.parametrize("steps", [[[5, 64, 0]], [[63, 1, 200]], [[65, 130, 128]], [[1, 60, 70], [1, 3, 57], [1, 1, 1], [70, 2, 66]]])
def test_store_and_load(gpu, steps, NKV, HS):
    """Codes and scales are the model's, to the bit; blocks of nobody stay, rows of nobody are not read or written."""
    nseq, cap = 3, 330
    c = Cache(gpu, nseq, cap, NKV, HS)
    g = gen(HS * 7 + len(steps))
    models = [(ref.Model(NKV, HS), ref.Model(NKV, HS)) for _ in range(nseq)]
    before = [t.clone() for t in c.parts()]
    keys = [0] * nseq
    for lens in steps:
        starts, rows = place_rows(lens)
        keys = [a + n for a, n in zip(keys, lens)]
        ld, off = NKV * HS + 3, 1
        k, v = (view(torch.full((off + rows * ld,), math.nan, device=DEV)[off:], rows, NKV, HS, ld) for _ in range(2))
        for b in range(nseq):
            at = slice(starts[b], starts[b] + lens[b])
            k[at] = rand(g, lens[b], NKV, HS) * torch.exp2(torch.randint(-4, 5, (lens[b], NKV, 1), generator=g, device=DEV).float())
            v[at] = rand(g, lens[b], NKV, HS, scale=0.3)
            for m, x in zip(models[b], (k, v)):
                m.store(x[at], keys[b])
        a = c.call(NKV, starts, lens, keys, rows, ldk=ld, ldv=ld)
        gpu.cache8_store(*c.parts(), k, v, a)
        out = [view(torch.full((off + rows * ld,), 7.0, device=DEV)[off:], rows, NKV, HS, ld) for _ in range(2)]
        gpu.cache8_load(*out, *c.parts(), a)
        gpu.synchronize()
        inside = torch.zeros(rows, dtype=torch.bool, device=DEV)
        for b in range(nseq):
            at = slice(starts[b], starts[b] + lens[b])
            inside[at] = True
            for name, m, o, sc in zip("kv", models[b], out, (c.ks, c.vs)):
                want = m.values()
                assert torch.equal(c.values(b, keys[b], name).cpu(), want), (b, name)
                nb = len(m.scales)
                assert torch.equal(sc[c.table[b, :nb].long()].cpu().double(), torch.stack(m.scales) if nb else sc[:0].cpu().double())
                assert torch.equal(o[at].double().cpu(), want[keys[b] - lens[b]:])
        assert all((o[~inside] == 7.0).all() for o in out)
    used = torch.zeros(c.nblocks, dtype=torch.bool, device=DEV)
    for b in range(nseq):
        used[c.table[b, :(keys[b] + 63) // 64].long()] = True
    assert all(torch.equal(x[~used], y[~used]) for x, y in zip(c.parts(), before))
    for b in range(nseq):  # and what lies behind a sequence's last key in its block
        n = keys[b] % 64
        if n:
            i = int(c.table[b, keys[b] // 64])
            assert torch.equal(c.k8[i, :, n:], before[0][i, :, n:])
            behind = ref.place()[n:].to(DEV)
            assert torch.equal(c.v8[i][..., behind], before[2][i][..., behind])


@pytest.mark.parametrize("nseq,lq,NKV,HS", [(40, 640, 8, 16), (100, 300, 8, 64), (70, 1000, 9, 33)])
def test_store_of_one_sequence_of_many_rows_among_many_of_one(gpu, nseq, lq, NKV, HS):
    """max_q is one sequence's: a call for all leaves what calls for each do."""
    cap = lq + 100
    lens, keys = [1 + b % 2 for b in range(nseq)], [2 + 11 * b % cap for b in range(nseq)]
    lens[nseq - 3], keys[nseq - 3], lens[3], lens[5], keys[5] = lq, cap, 0, 0, 0
    starts, rows = place_rows(lens)
    g = gen(nseq)
    k, v = rand(g, rows, NKV, HS), rand(g, rows, NKV, HS)
    c, d = (Cache(gpu, nseq, cap, NKV, HS, seed=5) for _ in "cd")
    gpu.cache8_store(*c.parts(), k, v, c.call(NKV, starts, lens, keys, rows))
    for b in range(nseq):
        a = d.gpu.Cache8(nseq=1, NH=NKV, NKV=NKV, HS=HS, rows_q=rows, max_q=lq, max_k=cap, nblocks=d.nblocks, q_start=ints([starts[b]]),
                         q_end=ints([starts[b] + lens[b]]), k_len=ints([keys[b]]), table=d.table[b:b + 1])
        gpu.cache8_store(*d.parts(), k, v, a)
    assert all(torch.equal(x, y) for x, y in zip(c.parts(), d.parts()))
    k2, v2 = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    gpu.cache8_load(k2, v2, *c.parts(), c.call(NKV, starts, lens, keys, rows))
    gpu.synchronize()
    for b in range(nseq):
        at = slice(starts[b], starts[b] + lens[b])
        for got, name in ((k2, "k"), (v2, "v")):
            assert torch.equal(got[at].double(), c.values(b, keys[b], name)[keys[b] - lens[b]:])
    used = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for b in range(nseq):
        used[starts[b]:starts[b] + lens[b]] = True
    assert (k2[~used] == 9.0).all() and (v2[~used] == 9.0).all()


def test_store_reports_rows_in_several_sequences(gpu):
    """As many blocks as a buffer of so many rows cannot touch: none is written outside its place."""
    nseq, lq, NKV, HS = 64, 640, 8, 16
    c = Cache(gpu, nseq, lq, NKV, HS)
    k = rand(gen(1), lq, NKV, HS)
    gpu.cache8_store(*c.parts(), k, k.clone(), c.call(NKV, [0] * nseq, [lq] * nseq, [lq] * nseq))
    with pytest.raises(gpu.UgkError, match="cache8_store"):
        gpu.synchronize()
    bad = Cache(gpu, nseq, lq, NKV, HS)
    keys = [lq] * nseq
    keys[50] = lq + 1
    lens = [1] * nseq
    lens[2] = lq
    starts, rows = place_rows(lens)
    k = rand(gen(1), rows, NKV, HS)
    gpu.cache8_store(*bad.parts(), k, k.clone(), bad.call(NKV, starts, lens, keys, rows))
    with pytest.raises(gpu.UgkError, match="cache8_store"):
        gpu.synchronize()


def one_block(gpu, values, NKV=1):
    """values: a list of rows of numbers, stored one call each; the codes and the scale of K and V."""
    HS = len(values[0])
    c = Cache(gpu, 1, 64, NKV, HS)
    for i, row in enumerate(values):
        x = torch.tensor(row, device=DEV).view(1, 1, HS)
        gpu.cache8_store(*c.parts(), x, x, c.call(1, [0], [1], [i + 1]))
    n = len(values)
    code = c.k8[c.table[0, 0].item(), 0, :n, :HS].cpu().long()
    vcode = c.v8[c.table[0, 0].item(), 0, :HS][:, ref.place()[:n].to(DEV)].T.cpu().long()
    assert torch.equal(code, vcode)
    i = c.table[0, 0].item()
    assert float(c.ks[i]) == float(c.vs[i])
    return code.tolist(), float(c.ks[i])


def test_scales_and_roundings_at_the_borders(gpu):
    big = 3.402823466e38
    for values, codes, scale in (
            ([[127.0, -127.0, 0.5, 1.5, 2.5, -0.5]], [[127, -127, 0, 2, 2, 0]], 1.0),
            ([[127.00001, 3.0, 1.0, -1.0, 5.0, 0.0]], [[64, 2, 0, 0, 2, 0]], 2.0),
            ([[0.0, -0.0]], [[0, 0]], 0.0),
            ([[0.0, 0.0], [1.0, 0.25]], [[0, 0], [64, 16]], 2.0 ** -6),
            ([[1e-44, 0.0]], [[0, 0]], 2.0 ** -126),
            ([[2.0 ** -120, 2.0 ** -126]], [[64, 1]], 2.0 ** -126),
            ([[big, 2.0 ** 121, -big]], [[127, 1, -127]], 2.0 ** 121),
            # older codes follow a larger scale, ties to even, and stay where a later row is smaller
            ([[1.0, 3.0 / 64, 1.0 / 64, 5.0 / 64]] + [[2.0, 0.0, 0.0, 0.0]] + [[0.5] * 4], [[32, 2, 0, 2], [64, 0, 0, 0], [16] * 4], 2.0 ** -5),
            ([[1.0, 1.0], [2.0 ** 20, 0.0]], [[0, 0], [64, 0]], 2.0 ** 14)):
        assert one_block(gpu, values) == (codes, scale), values
    gpu.synchronize()


def test_store_begins_a_block_anew(gpu):
    """A block that held large numbers has the scale of the new ones, whatever the shortened sequence left in it."""
    c = Cache(gpu, 1, 128, 1, 8)
    big, small = torch.full((70, 1, 8), 1000.0, device=DEV), torch.full((6, 1, 8), 0.5, device=DEV)
    gpu.cache8_store(*c.parts(), big, big, c.call(1, [0], [70], [70]))
    gpu.cache8_store(*c.parts(), small, small, c.call(1, [0], [6], [70]))  # k_len 64: rows 64 to 69 again
    assert float(c.ks[c.table[0, 1].long()]) == 2.0 ** -7
    gpu.cache8_store(*c.parts(), small, small, c.call(1, [0], [6], [66]))  # rows 60 to 65: the first block keeps its scale
    assert float(c.ks[c.table[0, 0].long()]) == 8.0 and float(c.ks[c.table[0, 1].long()]) == 2.0 ** -7
    assert torch.equal(c.values(0, 66, "k")[60:64].cpu(), torch.zeros(4, 1, 8, dtype=torch.float64))
    gpu.synchronize()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_numbers_that_8_bits_do_not_hold_are_reported(gpu, bad):
    c = Cache(gpu, 1, 64, 1, 4)
    x = torch.tensor([[1.0, bad, 2.0, 3.0]], device=DEV)
    gpu.synchronize()
    gpu.cache8_store(*c.parts(), x, x, c.call(1, [0], [1], [1]))
    with pytest.raises(gpu.UgkError, match="NaN or an infinity"):
        gpu.synchronize()
    gpu.synchronize()
    got = c.values(0, 1, "v").flatten().tolist()
    assert got == [1.0, 0.0, 2.0, 3.0] if math.isnan(bad) else got[1] == math.copysign(127 * 2.0 ** 121, bad)


def inside(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & ~(got.double() == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol.clamp(min=1e-300))[bad].nan_to_num(1e9).max()):.3g} of the bound"


def filled(gpu, nseq, cap, NKV, HS, keys, seed=3, size=None, **kw):
    c = Cache(gpu, nseq, cap, NKV, HS, seed=seed, **kw)
    g = gen(seed)
    starts, rows = place_rows(keys)
    k, v = rand(g, rows, NKV, HS), rand(g, rows, NKV, HS)
    if size:
        size(k, v)
    if sum(keys):
        gpu.cache8_store(*c.parts(), k, v, c.call(NKV, starts, keys, keys, rows))
    return c, g


def attend(gpu, c, NH, q, starts, lens, keys, rows, causal=True, weight=None, lse=True, pad=0, **kw):
    ldo = NH * c.HS + pad
    out = view(torch.full((rows * ldo,), 7.0, device=DEV), rows, NH, c.HS, ldo)
    L = torch.full((rows, NH), 7.0, device=DEV)
    a = c.call(NH, starts, lens, keys, rows, causal=causal, ldq=q.stride(0), ldo=ldo, **kw)
    gpu.cache8_attention(out, L if lse else None, q, *c.parts(), a, weight=weight)
    return out, L


def check(gpu, c, NH, q, starts, lens, keys, rows, causal=True, weigh=False, pad=0, scale=None, **kw):
    weight = torch.full(c.table.shape, 0.5, device=DEV) if weigh else None
    few = weigh or max(lens) * (NH // c.NKV) <= 64  # the rows whose weights may be whole numbers
    out, L = attend(gpu, c, NH, q, starts, lens, keys, rows, causal, weight, pad=pad, scale=scale, **kw)
    gpu.synchronize()
    s = c.HS ** -0.5 if scale is None else scale
    free = torch.ones(rows, dtype=torch.bool, device=DEV)
    for b in range(c.nseq):
        at = slice(starts[b], starts[b] + lens[b])
        free[at] = False
        if not lens[b]:
            if weigh:
                assert (weight[b] == 0.5).all()
            continue
        k, v = c.values(b, keys[b], "k"), c.values(b, keys[b], "v")
        o, l, w, tol, tol_l, tol_w = ref.attention(q[at], k, v, s, causal, few)
        inside(out[at], o, tol, f"out of {b}")
        inside(L[at], l, tol_l, f"lse of {b}")
        if weigh:
            n = len(w)
            inside(weight[b, :n], w + 0.5, tol_w + 2 * ref.U * (w + 0.5), f"weight of {b}")
            assert (weight[b, n:] == 0.5).all()
    assert (out[free] == 7.0).all() and (L[free] == 7.0).all()
    return out, L, weight


LENGTHS = {
    "token": ([1, 1, 1, 1], [1, 700, 64, 129]), "empty": ([1, 0, 3, 2], [0, 5, 0, 1]), "few": ([2, 4, 3, 1], [300, 5, 1030, 2]),
    "drafts": ([5, 8, 7, 1], [64, 8, 201, 65]), "later": ([20, 70, 5, 1], [7, 64, 0, 1]), "edge": ([63, 64, 65, 1], [63, 128, 65, 64]),
    "chunk": ([3, 129, 40, 128], [50, 333, 500, 128]), "prompt": ([300, 257, 1, 31], [300, 257, 1, 31]),
}


@pytest.mark.parametrize("NH,NKV,HS", [(1, 1, 64), (6, 2, 64), (4, 2, 128), (8, 1, 16), (4, 4, 50), (5, 1, 33), (2, 2, 1), (2, 1, 80), (3, 1, 96)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_attention(gpu, lens, NH, NKV, HS):
    lq, lk = LENGTHS[lens]
    c, g = filled(gpu, 4, 1030, NKV, HS, lk)
    starts, rows = place_rows(lq)
    ld = NH * HS + 5
    q = view(rand(g, 3 + rows * ld)[3:], rows, NH, HS, ld)
    for causal in (True, False):
        out, L, _ = check(gpu, c, NH, q, starts, lq, lk, rows, causal, pad=3)
        again, L2, _ = check(gpu, c, NH, q, starts, lq, lk, rows, causal, pad=3)
        assert torch.equal(out, again) and torch.equal(L, L2)


@pytest.mark.parametrize("lens,NH,NKV,HS", [("token", 6, 2, 64), ("empty", 4, 4, 64), ("few", 8, 2, 128), ("drafts", 3, 3, 50), ("drafts", 8, 1, 64),
                                            ("later", 6, 2, 80), ("edge", 4, 4, 32), ("chunk", 2, 2, 64)])
def test_weights_of_the_blocks(gpu, lens, NH, NKV, HS):
    lq, lk = LENGTHS[lens]
    c, g = filled(gpu, 4, 1030, NKV, HS, lk, ld=20)
    starts, rows = place_rows(lq)
    q = rand(g, rows, NH, HS, scale=2.0)
    for causal in (True, False):
        _, _, w = check(gpu, c, NH, q, starts, lq, lk, rows, causal, weigh=True)
        _, _, w2 = check(gpu, c, NH, q, starts, lq, lk, rows, causal, weigh=True)
        assert torch.equal(w, w2)


def test_defaults_of_the_call(gpu):
    """No offsets, lengths, table or lse: equal rows, full sequences, blocks in order."""
    nseq, cap, NH, NKV, HS = 3, 100, 4, 2, 64
    g = gen(5)
    n = nseq * 2
    k8 = torch.zeros(n, NKV, 64, HS, dtype=torch.int8, device=DEV)
    v8, ks = torch.zeros(n, NKV, HS, 64, dtype=torch.int8, device=DEV), torch.zeros(n, NKV, device=DEV)
    vs = torch.zeros_like(ks)
    k, v, q = rand(g, nseq * cap, NKV, HS), rand(g, nseq * cap, NKV, HS), rand(g, nseq * cap, NH, HS)
    a = gpu.Cache8(nseq=nseq, NH=NH, NKV=NKV, HS=HS, rows_q=nseq * cap, max_q=cap, max_k=cap, nblocks=n)
    gpu.cache8_store(k8, ks, v8, vs, k, v, a)
    out = torch.empty_like(q)
    gpu.cache8_attention(out, None, q, k8, ks, v8, vs, a)
    gpu.synchronize()
    uk, uv = ref.unpack(k8, ks, HS, False), ref.unpack(v8, vs, HS, True)
    for b in range(nseq):
        t, at = torch.tensor([2 * b, 2 * b + 1], device=DEV), slice(b * cap, (b + 1) * cap)
        o, _, _, tol, _, _ = ref.attention(q[at], ref.gather(uk, t, cap), ref.gather(uv, t, cap), HS ** -0.5, True, False)
        inside(out[at], o, tol, "out")


@pytest.mark.parametrize("lq", [1, 5, 40])
@pytest.mark.parametrize("what", ["large values of no weight", "small blocks", "near the top", "near the bottom", "large scores", "zeros", "rows apart"])
def test_digits(gpu, what, lq):
    """Sizes that a block must not pass on to another, or a row to the next."""
    NH, NKV, HS, n = 4, 2, 64, 500
    scale = HS ** -0.5

    def size(k, v):
        if what == "large values of no weight":
            k[100:164] = -k[100:164].abs()
            v[100:164] *= 2.0 ** 60
        elif what == "small blocks":
            v *= torch.exp2(-20.0 * (torch.arange(len(v), device=DEV) // 64))[:, None, None]
            k[:64] -= 3.0
        elif what == "near the top":
            v *= 2.0 ** 125 / v.abs().max()
        elif what == "near the bottom":
            v *= 2.0 ** -115
        elif what == "large scores":
            k *= 40.0
        elif what == "zeros":
            k[65:193] = 0.0
            v[1:129] = 0.0
    c, g = filled(gpu, 1, n, NKV, HS, [n], size=size)
    q = rand(g, lq, NH, HS)
    if what == "large values of no weight":
        q = q.abs() * 4 + 4
    if what == "rows apart":
        q *= torch.exp2(torch.randint(-60, 3, (lq, NH, 1), generator=g, device=DEV).float())
        q[0, 0] *= 2.0 ** -60
    check(gpu, c, NH, q, [0], [lq], [n], lq, scale=scale)
    check(gpu, c, NH, q, [0], [lq], [n], lq, scale=scale, weigh=True)


@pytest.mark.parametrize("lq", [2, 40])
def test_rows_that_are_no_numbers(gpu, lq):
    """A row of q with an infinity or NaN, or whose scores overflow, is NaN, and no other row is touched by it."""
    NH, NKV, HS, n = 2, 1, 64, 200
    c, g = filled(gpu, 1, n, NKV, HS, [n])
    q = rand(g, lq, NH, HS)
    clean, L0 = attend(gpu, c, NH, q, [0], [lq], [n], lq)
    bad = q.clone()
    bad[0, 1, 3], bad[1, 0, 5] = math.nan, math.inf
    out, L = attend(gpu, c, NH, bad, [0], [lq], [n], lq)
    hit = torch.zeros(lq, NH, dtype=torch.bool, device=DEV)
    hit[0, 1] = hit[1, 0] = True
    assert out[hit].isnan().all() and L[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(L[~hit], L0[~hit])
    big = q.clone()
    big[0, 0] = 3e38 * torch.sign(c.values(0, n, "k")[0, 0].float())  # scores beyond the range, some of them above
    out, L = attend(gpu, c, NH, big, [0], [lq], [n], lq, scale=1.0)
    assert out[0, 0].isnan().all() and L[0, 0].isnan() and out[1].isfinite().all()
    down = q.clone()
    down[0, 0] = -3e38
    same, s = filled(gpu, 1, n, NKV, HS, [n], size=lambda k, v: k.abs_())
    out, L = attend(gpu, same, NH, down, [0], [lq], [n], lq, scale=1.0)  # all of them below: no weight at all
    assert (out[0, 0] == 0).all() and L[0, 0] == -math.inf and out[1].isfinite().all()
    out, L = attend(gpu, same, NH, q, [0], [lq], [n], lq, scale=0.0)  # the mean
    assert torch.allclose(out[0, 0].double(), same.values(0, n, "v")[:n - lq + 1, 0].mean(0), atol=1e-6)
    gpu.synchronize()


@pytest.mark.parametrize("cap", [300, 2500])
@pytest.mark.parametrize("lq", [1, 6, 20])
def test_weights_of_a_row_that_is_no_number(gpu, lq, cap):
    """The blocks that it sees get NaN; other sequences' get what they would."""
    NH, NKV, HS = 4, 2, 64
    keys = [cap - 70, cap, 90]
    c, g = filled(gpu, 3, cap, NKV, HS, keys)
    starts, rows = place_rows([lq] * 3)
    q = rand(g, rows, NH, HS)
    want, got = (torch.zeros(c.table.shape, device=DEV) for _ in "wg")
    attend(gpu, c, NH, q, starts, [lq] * 3, keys, rows, weight=want)
    q[starts[1], 3, 9] = math.nan
    attend(gpu, c, NH, q, starts, [lq] * 3, keys, rows, weight=got)
    gpu.synchronize()
    seen = -(-(keys[1] - lq + 1) // 64)  # of the sequence's first row
    assert got[1, :seen].isnan().all() and not got[1, seen:].isnan().any()
    assert torch.equal(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("lq", [1, 3, 40])
def test_what_lies_outside_does_not_matter(gpu, lq):
    """Codes behind the last key, blocks of others, scales of others, q rows of nobody: the same bits whatever they are."""
    NH, NKV, HS, keys = 4, 2, 64, [100, 65]
    c, g = filled(gpu, 2, 300, NKV, HS, keys)
    starts, rows = place_rows([lq, lq])
    q = rand(g, rows, NH, HS)
    first = [t.clone() for t in attend(gpu, c, NH, q, starts, [lq] * 2, keys, rows)]
    used = torch.zeros(c.nblocks, dtype=torch.bool, device=DEV)
    for b, n in enumerate(keys):
        used[c.table[b, :(n + 63) // 64].long()] = True
        i = int(c.table[b, n // 64])
        c.k8[i, :, n % 64:] = -128
        c.v8[i][..., ref.place()[n % 64:].to(DEV)] = -128
        c.table[b, (n + 63) // 64:] = -5  # blocks that are not there yet
    c.k8[~used], c.v8[~used], c.ks[~used], c.vs[~used] = 127, 127, math.nan, math.inf
    free = torch.ones(rows, dtype=torch.bool, device=DEV)
    for s in starts:
        free[s:s + lq] = False
    q[free] = math.nan
    second = attend(gpu, c, NH, q, starts, [lq] * 2, keys, rows)
    gpu.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_blocks_and_lengths_out_of_range_are_reported(gpu):
    NH, NKV, HS = 2, 2, 64
    c, g = filled(gpu, 2, 200, NKV, HS, [150, 200])
    k, out = rand(g, 4, NKV, HS), torch.empty(4, NH, HS, device=DEV)
    load = [torch.empty(4, NKV, HS, device=DEV) for _ in range(2)]
    gpu.synchronize()

    def each(**kw):
        kw = {**dict(keys=[150, 200], starts=[0, 2], lens=[2, 2]), **kw}
        extra = {n: kw.pop(n) for n in list(kw) if n not in ("keys", "starts", "lens")}
        a = c.call(NH, kw["starts"], kw["lens"], kw["keys"], 4, **{"max_q": 2, **extra})
        held = [t.clone() for t in c.parts()]
        for name, call in (("store", lambda: gpu.cache8_store(*c.parts(), k, k, a)), ("load", lambda: gpu.cache8_load(*load, *c.parts(), a)),
                           ("attention", lambda: gpu.cache8_attention(out, None, k, *c.parts(), a))):
            call()
            with pytest.raises(gpu.UgkError, match="cache8_" + name):
                gpu.synchronize()
            gpu.synchronize()
        return held
    each(keys=[150, 201])
    each(keys=[-1, 100])
    each(starts=[0, 3])
    each(starts=[-1, 2])
    each(lens=[3, 1])
    table = c.table.clone()
    for bad in (-1, c.nblocks, 2 ** 31 - 1, -2 ** 31):
        c.table[1, 3] = bad  # the block that the last rows are in
        held = each()
        c.table.copy_(table)
        others = torch.ones(c.nblocks, dtype=torch.bool, device=DEV)
        others[c.table[0, 2].long()] = False
        assert all(torch.equal(x[others], y[others]) for x, y in zip(c.parts(), held))
    gpu.cache8_store(*c.parts(), k, k, c.call(NH, [0, 2], [2, 2], [1, 100], 4))  # two rows for one key
    with pytest.raises(gpu.UgkError, match="cache8_store"):
        gpu.synchronize()
    assert torch.equal(c.values(0, 1, "k")[0].float().round(decimals=1).isfinite(), torch.ones(NKV, HS, dtype=torch.bool, device=DEV))
    gpu.synchronize()


def test_a_missing_block_is_as_if_its_keys_were_not_there(gpu):
    NH, NKV, HS, n = 2, 1, 64, 256
    for lq in (1, 40):
        c, g = filled(gpu, 1, n, NKV, HS, [n])
        q = rand(g, lq, NH, HS)
        whole = c.table.clone()
        c.table[0, 1] = -1
        out, L = attend(gpu, c, NH, q, [0], [lq], [n], lq)
        with pytest.raises(gpu.UgkError, match="cache8_attention"):
            gpu.synchronize()
        c.table = whole[:, [0, 2, 3]].contiguous()
        o, l, _, tol, tol_l, _ = ref.attention(q, c.values(0, 192, "k"), c.values(0, 192, "v"), HS ** -0.5, True, lq == 1)
        inside(out, o, tol, "out")
        inside(L, l, tol_l, "lse")


def test_offsets_beyond_32_bits(gpu):
    """Blocks whose codes begin 2^31 bytes and more into the cache, rows of q 2^31 bytes and more into theirs."""
    NKV, HS, n = 2, 128, 150
    nblocks = (1 << 31) // (NKV * 64 * HS) + 70
    k8 = torch.zeros(nblocks, NKV, 64, HS, dtype=torch.int8, device=DEV)
    v8, ks = torch.zeros(nblocks, NKV, HS, 64, dtype=torch.int8, device=DEV), torch.zeros(nblocks, NKV, device=DEV)
    vs = torch.zeros_like(ks)
    g, ld = gen(2), 1 << 24
    table = ints([[nblocks - 1, 3, nblocks - 60]])
    k, v = rand(g, n, NKV, HS), rand(g, n, NKV, HS)
    kw = dict(nseq=1, NH=4, NKV=NKV, HS=HS, max_k=n, nblocks=nblocks, table=table)
    gpu.cache8_store(k8, ks, v8, vs, k, v, gpu.Cache8(rows_q=n, max_q=n, **kw))
    for lq in (3, 40):
        buf = torch.empty(lq * ld, device=DEV)
        q = view(buf, lq, 4, HS, ld)
        q.copy_(rand(g, lq, 4, HS))
        out = torch.empty(lq, 4, HS, device=DEV)
        gpu.cache8_attention(out, None, q, k8, ks, v8, vs, gpu.Cache8(rows_q=lq, max_q=lq, ldq=ld, **kw))
        gpu.synchronize()
        uk, uv = (ref.unpack(x[table[0].long()], y[table[0].long()], HS, z) for x, y, z in ((k8, ks, False), (v8, vs, True)))
        t = torch.arange(3, device=DEV)
        o, _, _, tol, _, _ = ref.attention(q, ref.gather(uk, t, n), ref.gather(uv, t, n), HS ** -0.5, True, lq == 3)
        inside(out, o, tol, "out")
        del buf, q


@pytest.mark.parametrize("nseq,lq,NH,NKV,HS,cap", [(1, 1, 8, 1, 128, 9000), (1, 8, 4, 1, 64, 5000), (40, 1, 4, 4, 64, 700), (2, 33, 1, 1, 128, 4100),
                                                   (3, 200, 4, 2, 128, 2300), (70, 2, 2, 2, 16, 65)])
def test_split_key_axes(gpu, nseq, lq, NH, NKV, HS, cap):
    g = gen(cap)
    keys = [max(lq, cap - 37 * b) for b in range(nseq)]
    c, _ = filled(gpu, nseq, cap, NKV, HS, keys, seed=cap)
    starts, rows = place_rows([lq] * nseq, gap=0, tail=0)
    q = rand(g, rows, NH, HS)
    check(gpu, c, NH, q, starts, [lq] * nseq, keys, rows)
    if lq * NH // NKV <= 256:
        check(gpu, c, NH, q, starts, [lq] * nseq, keys, rows, weigh=True)


@pytest.mark.parametrize("lq,NH,NKV,HS", [(1, 2, 2, 16), (3, 4, 1, 64), (7, 4, 2, 33), (40, 2, 1, 64)])
@pytest.mark.parametrize("nseq", [5, 64, 131])
def test_many_sequences_of_very_different_lengths(gpu, nseq, lq, NH, NKV, HS):
    """Parts dealt out by what the sequences hold: some have no rows, some no keys, few have almost all of them."""
    g = torch.Generator().manual_seed(nseq + lq)
    cap = 2500
    keys = [0 if r < 0.1 else int(cap ** r) for r in torch.rand(nseq, generator=g).tolist()]
    keys[-1] = cap
    lens = [0 if r < 0.2 else max(1, int(lq * r)) for r in torch.rand(nseq, generator=g).tolist()]
    lens[-1] = lens[0] = lq
    c, gg = filled(gpu, nseq, cap, NKV, HS, keys, seed=nseq)
    starts, rows = place_rows(lens)
    q = rand(gg, rows, NH, HS)
    out, L, _ = check(gpu, c, NH, q, starts, lens, keys, rows, max_q=lq)
    again, L2, _ = check(gpu, c, NH, q, starts, lens, keys, rows, max_q=lq)
    assert torch.equal(out, again) and torch.equal(L, L2)
    check(gpu, c, NH, q, starts, lens, keys, rows, causal=False, max_q=lq)
    if lq * NH // NKV <= 256:
        check(gpu, c, NH, q, starts, lens, keys, rows, weigh=True, max_q=lq)


@pytest.mark.parametrize("nseq,lq,NH,NKV,HS,cap,equal", [(100, 1, 16, 16, 16, 2200, False), (40, 1, 16, 16, 16, 2600, True),
                                                         (3, 300, 3, 1, 80, 3000, False), (20, 9, 14, 2, 33, 2100, False),
                                                         (6, 130, 5, 1, 128, 4500, False), (1, 4, 1, 1, 64, 2113, True)])
def test_blocks_dealt_out_in_equal_shares(gpu, nseq, lq, NH, NKV, HS, cap, equal):
    """More groups of rows than workgroups, groups that are each a workgroup's, heads of groups that are no power of two, rows
    before the first key, many short sequences in one workgroup."""
    g = torch.Generator().manual_seed(cap + nseq)
    keys = [cap if equal else max(1, int(cap ** r)) for r in torch.rand(nseq, generator=g).tolist()]
    keys[-1] = cap
    lens = [max(1, lq - b % 3) for b in range(nseq)]
    c, gg = filled(gpu, nseq, cap, NKV, HS, keys, seed=nseq)
    starts, rows = place_rows(lens)
    q = rand(gg, rows, NH, HS)
    check(gpu, c, NH, q, starts, lens, keys, rows, max_q=lq)
    check(gpu, c, NH, q, starts, lens, keys, rows, causal=False, max_q=lq)
    if lq * NH // NKV <= 256:
        check(gpu, c, NH, q, starts, lens, keys, rows, weigh=True, max_q=lq)


@pytest.mark.parametrize("lq,NH,NKV,HS", [(5, 4, 1, 128), (17, 1, 1, 64), (19, 2, 2, 33), (6, 3, 1, 96), (20, 2, 1, 64), (35, 1, 1, 16), (33, 2, 1, 80)])
@pytest.mark.parametrize("cap", [200, 2500])
def test_groups_of_rows_that_end_in_a_few(gpu, cap, lq, NH, NKV, HS):
    """A few rows and heads more than 16, and with weights than 32."""
    keys, lens = [cap, 3, cap // 2, 64], [lq, lq, lq - 1, 1]
    c, g = filled(gpu, 4, cap, NKV, HS, keys, seed=cap + lq)
    starts, rows = place_rows(lens)
    q = rand(g, rows, NH, HS)
    for causal in (True, False):
        check(gpu, c, NH, q, starts, lens, keys, rows, causal=causal)
        check(gpu, c, NH, q, starts, lens, keys, rows, causal=causal, weigh=True)


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("lq,NH,NKV,HS,cap", [(640, 1, 1, 64, 500), (200, 3, 1, 33, 2300), (36, 14, 2, 16, 300), (9, 4, 1, 128, 2500), (5000, 2, 1, 16, 5100)])
def test_one_sequence_of_many_rows_among_many_of_one(gpu, lq, NH, NKV, HS, cap, weigh):
    """max_q is one sequence's: most groups of rows are not there."""
    if weigh and lq * NH // NKV > 256:
        return
    nseq = 40
    lens, keys = [1] * nseq, [1 + 7 * b % cap for b in range(nseq)]
    lens[17], keys[17], lens[3], keys[3], lens[39] = lq, cap, 0, 0, 0
    c, g = filled(gpu, nseq, cap, NKV, HS, keys)
    starts, rows = place_rows(lens)
    q = rand(g, rows, NH, HS)
    check(gpu, c, NH, q, starts, lens, keys, rows, weigh=weigh)


@pytest.mark.parametrize("lq,weigh", [(320, False), (48, False), (48, True)])
def test_rows_in_several_sequences_are_reported(gpu, lq, weigh):
    """64 sequences of the same rows, whose groups are more than a buffer of so many rows has: nothing is computed."""
    nseq, cap, HS = 64, 2200, 16
    c, g = filled(gpu, nseq, cap, 1, HS, [cap] * nseq)
    q, out = rand(g, lq, 1, HS), torch.full((lq, 1, HS), 7.0, device=DEV)
    weight = torch.zeros(nseq, c.table.shape[1], device=DEV) if weigh else None
    gpu.cache8_attention(out, None, q, *c.parts(), c.call(1, [0] * nseq, [lq] * nseq, [cap] * nseq), weight=weight)
    with pytest.raises(gpu.UgkError, match="cache8_attention"):
        gpu.synchronize()
    assert (out == 7.0).all() and (not weigh or not weight.any())


@pytest.mark.parametrize("lq,NH,NKV,HS", [(1, 2, 1, 64), (7, 6, 3, 33), (50, 3, 1, 16)])
def test_a_padded_batch(gpu, lq, NH, NKV, HS):
    """Few of many sequences have rows."""
    nseq, cap = 333, 2200
    lens, keys = [0] * nseq, [0] * nseq
    for b, n in ((2, 2200), (3, 40), (66, 1), (67, 700), (68, 64), (200, 2100), (331, 1500)):
        lens[b], keys[b] = lq, n
    c, g = filled(gpu, nseq, cap, NKV, HS, keys)
    starts, rows = place_rows(lens, gap=0)
    q = rand(g, rows, NH, HS)
    check(gpu, c, NH, q, starts, lens, keys, rows)
    if lq * NH // NKV <= 256:
        check(gpu, c, NH, q, starts, lens, keys, rows, weigh=True)


def test_many_groups_of_rows_in_a_sequence(gpu):
    """More than 64 workgroups' rows in one sequence, whose key axis is cut all the same."""
    NH, NKV, HS, lq, n = 8, 1, 16, 1100, 2400
    c, g = filled(gpu, 2, n, NKV, HS, [n, 70])
    starts, rows = place_rows([lq, 3])
    q = rand(g, rows, NH, HS)
    check(gpu, c, NH, q, starts, [lq, 3], [n, 70], rows)


@pytest.mark.parametrize("lq", [1, 5, 40])
def test_scores_far_below_zero(gpu, lq):
    """Blocks of which a row sees nothing, next to scores of -1,000 and less."""
    NH, NKV, HS, n = 2, 1, 64, 450  # the rows lie on both sides of the border at 448
    c, g = filled(gpu, 1, n, NKV, HS, [n], size=lambda k, v: k.abs_().add_(1.0))
    q = -rand(g, lq, NH, HS).abs() - 2.0
    check(gpu, c, NH, q, [0], [lq], [n], lq, scale=8.0)
    check(gpu, c, NH, q, [0], [lq], [n], lq, scale=8.0, weigh=True)
    check(gpu, c, NH, -q, [0], [lq], [n], lq, scale=-8.0)


def test_captured_and_on_another_stream(gpu):
    """Store, attention with weights and eviction in a graph, replayed between eager calls on another stream."""
    NH, NKV, HS, cap, nseq = 4, 2, 64, 500, 3
    keys = [100, 64, 333]
    c, g = filled(gpu, nseq, cap, NKV, HS, keys)
    starts, rows = place_rows([2] * nseq, gap=0, tail=0)
    x, out = rand(g, rows, NH + 2 * NKV, HS), torch.empty(rows, NH, HS, device=DEV)
    weight, dropped = torch.zeros(c.table.shape, device=DEV), ints([0] * nseq)
    ld = (NH + 2 * NKV) * HS
    lens = ints(keys)
    a = c.call(NH, starts, [2] * nseq, keys, rows, k_len=lens, ldq=ld, ldk=ld, ldv=ld)
    a2 = [t.clone() for t in (c.table, lens)]

    def step():
        weight.zero_()
        gpu.cache8_store(*c.parts(), x[:, NH:], x[:, NH + NKV:], a)
        gpu.cache8_attention(out, None, x, *c.parts(), a, weight=weight)
        gpu.cache8_evict(c.table, lens, weight, dropped, c.table, lens, weight, nseq, c.table.shape[1], 4, 1, 1)
    state = [t.clone() for t in c.parts()]

    def reset():
        for t, s in zip((*c.parts(), c.table, lens), (*state, *a2)):
            t.copy_(s)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gpu.set_stream(s.cuda_stream)
        try:
            step()
            want = [t.clone() for t in (out, weight, dropped, c.table, lens, *c.parts())]
            reset()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                step()
            for n in range(3):
                reset()
                out.fill_(n)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                for t, w in zip((out, weight, dropped, c.table, lens, *c.parts()), want):
                    assert torch.equal(t, w), n
                reset()
                step()
                torch.cuda.synchronize()
                assert torch.equal(out, want[0])
        finally:
            s.synchronize()
            gpu.set_stream(None)
    assert dropped.tolist() == [0, 0, 2]


@pytest.mark.parametrize("lq,NH,weigh", [(1, 2, True), (6, 8, True), (70, 4, False)])
def test_captured_with_lengths_that_change(gpu, lq, NH, weigh):
    """A graph's replays take the lengths, rows and blocks that the tensors hold then, and share out the work anew."""
    NKV, HS, cap, nseq = 2, 64, 2600, 5
    c, g = filled(gpu, nseq, cap, NKV, HS, [cap] * nseq)
    starts, rows = place_rows([lq] * nseq)
    q = rand(g, rows, NH, HS)
    out, lse = torch.empty(rows, NH, HS, device=DEV), torch.empty(rows, NH, device=DEV)
    weight = torch.zeros(c.table.shape, device=DEV) if weigh else None
    lens, end = ints([cap] * nseq), ints([a + lq for a in starts])
    a = c.call(NH, starts, [lq] * nseq, [cap] * nseq, rows, k_len=lens, q_end=end)

    def step():
        if weigh:
            weight.zero_()
        gpu.cache8_attention(out, lse, q, *c.parts(), a, weight=weight)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gpu.set_stream(s.cuda_stream)
        try:
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                step()
            for n, keys in enumerate(([cap, 1, 700, 64, 0], [lq] * nseq, [2048, 2049, cap, 3, 1], [cap] * nseq)):
                lens.copy_(ints(keys))
                end.copy_(ints([x + lq - (b + n) % 2 * (lq // 2) for b, x in enumerate(starts)]))
                c.table.copy_(c.table.roll(n, 0))
                for t in (out, lse):
                    t.fill_(5.0)
                step()
                want = [t.clone() for t in (out, lse, weight) if t is not None]
                for t in (out, lse):
                    t.fill_(5.0)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(t, w) for t, w in zip([t for t in (out, lse, weight) if t is not None], want)), n
        finally:
            s.synchronize()
            gpu.set_stream(None)
    check(gpu, c, NH, q, starts, [lq] * nseq, [cap] * nseq, rows, weigh=weigh)


def test_tensors_too_small_are_refused(gpu):
    c, g = filled(gpu, 2, 200, 2, 64, [150, 200])
    q, out = rand(g, 2, 4, 64), torch.empty(2, 4, 64, device=DEV)
    kw = dict(starts=[0, 1], lens=[1, 1], keys=[150, 200])
    call = lambda a, **t: gpu.cache8_attention(t.get("out", out), t.get("lse"), t.get("q", q), t.get("k8", c.k8), t.get("ks", c.ks), c.v8, c.vs, a, weight=t.get("weight"))  # noqa: E731
    a = c.call(4, **kw)
    call(a)
    for bad in (dict(out=out[:1].clone()), dict(lse=torch.empty(7, device=DEV)), dict(q=q[:1].clone()), dict(k8=c.k8[1:].clone()), dict(ks=c.ks[1:].clone()),
                dict(weight=torch.zeros(2, 3, device=DEV))):
        with pytest.raises(ValueError):
            call(a, **bad)
    for bad in (dict(k8=c.k8.float()), dict(ks=c.ks.double()), dict(q=q.half())):
        with pytest.raises(TypeError):
            call(a, **bad)
    with pytest.raises(ValueError, match="table"):
        c.call(4, table=c.table[:1].contiguous(), ld_table=4, **kw)
    with pytest.raises(ValueError, match="k_len"):
        c.call(4, k_len=ints([5]), **kw)
    a.nseq = 3
    with pytest.raises(ValueError, match="nseq"):
        call(a)
    a.nseq, a.ld_table = 2, 5
    with pytest.raises(ValueError, match="table"):
        call(a)
    with pytest.raises(gpu.UgkError, match="256 rows"):
        call(c.call(4, [0, 1], [1, 1], [150, 200], 400, max_q=129), q=torch.zeros(400, 4, 64, device=DEV), out=torch.zeros(400, 4, 64, device=DEV),
             weight=torch.zeros(2, 4, device=DEV))
    gpu.synchronize()


def test_workspace_of_the_caller(gpu):
    """What cuts the key axis fits a workspace of a config's size; the weights' memory is refused where it does not."""
    NH, NKV, HS = 12, 12, 64
    cfg = gpu.Config(B=4, T=1024, C=768, V=50, NH=NH, maxT=1024, L=1)
    n = gpu.workspace_bytes(cfg)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=DEV)
    at = (-ws.data_ptr()) % 256
    try:
        gpu.set_workspace(ws[at:at + n], cfg)
        for nseq, lq, cap in ((4, 1, 1024), (1, 1, 16384), (32, 8, 1000), (1, 40, 9000), (2, 300, 1000)):
            c, g = filled(gpu, nseq, cap, NKV, HS, [cap] * nseq)
            q = rand(g, nseq * lq, NH, HS)
            starts = [b * lq for b in range(nseq)]
            out, _ = attend(gpu, c, NH, q, starts, [lq] * nseq, [cap] * nseq, nseq * lq)
            o, _, _, tol, _, _ = ref.attention(q[:lq], c.values(0, cap, "k"), c.values(0, cap, "v"), HS ** -0.5, True, lq <= 32)
            inside(out[:lq], o, tol, "out")
        # 8 bytes for each of 61,440 rows and heads and 256 blocks: 126 MB, where the config has 80
        c, g = filled(gpu, 256, 16384, 1, 16, [100] * 256)
        q = rand(g, 256 * 20, 12, 16)
        with pytest.raises(gpu.UgkError, match="attention") as e:
            attend(gpu, c, 12, q, [20 * b for b in range(256)], [20] * 256, [100] * 256, 5120, weight=torch.zeros(c.table.shape, device=DEV))
        assert e.value.status == 3
        gpu.synchronize()
    finally:
        gpu.set_workspace(None, cfg)


# ---- eviction -----------------------------------------------------------------------

def check_evict(gpu, table, lens, weight, keep, first, recent, alias=False):
    nseq, ld = table.shape
    t, n, w = table.to(DEV), lens.to(DEV), weight.to(DEV)
    to = (t, n, w) if alias else (torch.full_like(t, -9), torch.full_like(n, -9), torch.full_like(w, -9.0))
    dropped = torch.full((nseq,), -9, dtype=torch.int32, device=DEV)
    gpu.cache8_evict(*to, dropped, t, n, w, nseq, ld, keep, first, recent)
    gpu.synchronize()
    rows, ws = table.tolist(), weight.tolist()
    for b in range(nseq):
        wt, wn, ww, wd = ref.evict(rows[b], int(lens[b]), ws[b], keep, first, recent)
        assert to[0][b].tolist() == wt and int(to[1][b]) == wn and int(dropped[b]) == wd, b
        got = to[2][b].cpu()
        want = torch.tensor(ww, dtype=torch.float32)
        assert torch.equal(got.nan_to_num(-3.0), want.nan_to_num(-3.0)), b


@pytest.mark.parametrize("ld", [1, 2, 63, 64, 65, 700, 1024, 1025, 4096, 5000, 16384])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(gpu, kind, ld):
    g = torch.Generator().manual_seed(ld)
    nseq = 5
    table = torch.stack([torch.randperm(ld * 2, generator=g)[:ld] for _ in range(nseq)]).int()
    lens = torch.randint(0, ld * 64 + 1, (nseq,), generator=g, dtype=torch.int32)
    lens[0] = ld * 64
    weight = torch.rand(nseq, ld, generator=g) * torch.exp(4 * torch.randn(nseq, ld, generator=g))
    if kind == "ties":
        weight = torch.randint(0, 3, (nseq, ld), generator=g).float()
    if kind == "odd":  # negative ones, zeros of both signs, infinities, NaN
        pick = torch.randint(0, 8, (nseq, ld), generator=g)
        odd = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -1.0, 1e-42, 3e38])
        weight = torch.where(torch.rand(nseq, ld, generator=g) < 0.7, odd[pick], weight)
    for keep, first, recent in ((1, 0, 1), (max(2, ld // 2), 1, 1), (max(3, ld // 3), 2, 1), (max(9, ld - 1), 4, 5), (ld + 5, 0, 1)):
        check_evict(gpu, table, lens, weight, keep, first, recent)
    check_evict(gpu, table, lens, weight, max(2, ld // 4), 1, 1, alias=True)


def test_evict_reports_lengths_out_of_range(gpu):
    table, w = ints([[0, 1, 2], [3, 4, 5]]), torch.ones(2, 3, device=DEV)
    for bad, n in ((193, 192), (-1, 0), (2 ** 31 - 1, 192)):
        to = [torch.empty_like(table), ints([0, 0]), torch.empty_like(w), ints([0, 0])]
        gpu.cache8_evict(*to, table, ints([100, bad]), w, 2, 3, 2)
        with pytest.raises(gpu.UgkError, match="cache8_evict"):
            gpu.synchronize()
        assert to[1].tolist() == [100, max(0, n - 64)] and sorted(to[0][1].tolist()) == [3, 4, 5]
    gpu.synchronize()


def test_attention_over_what_an_eviction_leaves(gpu):
    """The kept blocks' keys, in their order, and the store behind them grows into the dropped ones."""
    NH, NKV, HS, cap, n = 2, 1, 64, 512, 500
    c, g = filled(gpu, 1, cap, NKV, HS, [n])
    weight = torch.tensor([[5.0, 1.0, 4.0, 0.5, 9.0, 2.0, 3.0, 0.0]], device=DEV)
    lens, dropped = ints([n]), ints([0])
    k, v = c.values(0, n, "k"), c.values(0, n, "v")
    old = c.table.clone()
    gpu.cache8_evict(c.table, lens, weight, dropped, c.table, lens, weight, 1, 8, 5, 1, 1)
    assert dropped.tolist() == [3] and lens.tolist() == [n - 192]
    assert c.table[0].tolist() == old[0, [0, 2, 4, 6, 7, 1, 3, 5]].tolist()
    stay = torch.cat([torch.arange(64 * j, min(64 * j + 64, n), device=DEV) for j in (0, 2, 4, 6, 7)])
    q = rand(g, 1, NH, HS)
    out, L = attend(gpu, c, NH, q, [0], [1], lens.tolist(), 1)
    o, l, _, tol, tol_l, _ = ref.attention(q, k[stay], v[stay], HS ** -0.5, True, True)
    inside(out, o, tol, "out")
    inside(L, l, tol_l, "lse")
    m = n - 192
    more = rand(g, 60, NKV, HS)
    gpu.cache8_store(*c.parts(), more, more, c.call(NH, [0], [60], [m + 60]))
    gpu.synchronize()
    assert torch.equal(c.values(0, m, "k")[:256], k[stay][:256])
    late = c.values(0, m + 60, "v")
    s = c.vs[c.table[0].long()].double()
    assert ((late[m:] - more.double()).abs() <= 0.5 * s[(torch.arange(m, m + 60, device=DEV) // 64)][:, :, None]).all()
