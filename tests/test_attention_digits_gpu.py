"""GPU: the digits of attention's results where the sizes of what goes into them differ: a large value of little weight,
keys that hardly a row weighs, keys, values, queries and gradients whose size changes from row to row, scores of -infinity.

The bounds, from 64 bits, with u = 2^-24. A row of q, k, v or dout of one head enters products to 2^-23 of each element
(two 11-bit halves) and 2^-31 of its own largest (a tile is held at one scale only where its rows' largest are within
2^6 of each other, so a row's largest is 2^7 or more in the halves' units, and 2^-25 the error of a half there); the
omitted product of the two lower parts is 2^-22 of the product. Sums of HS such products are of 3 HS terms in 32 bits.
So a score is off by

    es = |scale| ((3 HS + 16) u sum |q k| + HS 2^-29 max|q| max|k|),

its exponential by a factor of es and, for the rounding of the exponent, 4 u (|s| + |lse| + 4) more, and a row's sum of
them by the mean of that over its weights; weights and results below 2^-126, the least number with 24 bits, by that (a
product of 2^-105 and 2^-90 is 0 in 32 bits). Weights, and the
score gradients of the backward, are held to two halves next to the largest contribution (weight times the row's
largest) that the row or the key sees. In the forward that contribution is 2^14 or more in the halves' units (P of 2^7 or
more times a value of 2^7 or more at the tile's scale), where another's P is off by 2^-25, times a value below
2^15: 2^-24 of it for each term, here 2^-23. In the backward the largest P or dS is 2^12 or more, times 2^7: 2^-29, here 2^-28.
"""
import math

import pytest
import torch

import att_ref
from att_ref import Seqs
from test_attention_gpu import DEV, Call, inside, rand

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def top(t):
    return t.abs().amax(-1) if t.shape[0] else t.new_zeros(t.shape[:-1])


def results(c, lse=None, out=None):
    """out, lse, dq, dk, dv in 64 bits with their bounds; the gradients are those of the given out and lse."""
    s, HS, G = c.s, c.HS, c.NH // c.NKV
    w = {}
    for name, t in (("out", c.q), ("lse", c.q[:, :, 0]), ("dq", c.q), ("dk", c.k), ("dv", c.k)):
        w[name] = (torch.zeros(t.shape, dtype=torch.float64, device=DEV), torch.full(t.shape, 2.0 ** -126, dtype=torch.float64, device=DEV))
    for b in range(len(s.lq)):
        for h in range(c.NH):
            rq, rk, q, k, v = att_ref._pieces(s, b, h, G, c.q, c.k, c.v)
            n, g = k.shape[0], c.dout[rq, h].double()
            ok = att_ref.allowed(q.shape[0], n, c.causal, DEV)
            S = (q @ k.T * c.scale).masked_fill(~ok, -math.inf)
            es = abs(c.scale) * ((3 * HS + 16) * U * (q.abs() @ k.abs().T) + HS * 2.0 ** -29 * top(q)[:, None] * top(k)[None])
            L = torch.logsumexp(S, 1)
            none = L == -math.inf
            weigh = lambda L: torch.where(S == -math.inf, 0.0, torch.exp(S - torch.where(none, 0.0, L)[:, None]))  # noqa: E731
            rel = lambda P: torch.where(P > 0, es + 4 * U * (S.abs() + L.abs()[:, None] + 4), 0.0)  # noqa: E731
            P = weigh(L)
            r, least = rel(P), 2.0 ** -126 * ok
            mean = (P * r + least).sum(1)
            w["out"][0][rq, h] = torch.where(P > 0, P, 0.0) @ torch.where(v.isfinite(), v, 0.0)
            w["lse"][0][rq, h] = L
            w["lse"][1][rq, h] += torch.where(none, 0.0, mean + (n + 16) * U + 4 * U * L.abs())
            biggest = (P * top(v)[None]).amax(1, keepdim=True) if n else 0.0
            w["out"][1][rq, h] += (P * (r + mean[:, None] + (2 * n + 32) * U) + least) @ v.abs() + \
                (P @ top(v))[:, None] * 2.0 ** -30 + n * 2.0 ** -23 * biggest
            if lse is None:
                continue
            o, L = out[rq, h].double(), lse[rq, h].double()
            P = weigh(L)
            r = rel(P)
            D, Da = (g * o).sum(1, keepdim=True), (g * o).abs().sum(1, keepdim=True)
            dP, dPa = g @ v.T, g.abs() @ v.abs().T
            dS = P * (dP - D) * c.scale
            eS = abs(c.scale) * least * (dPa + Da) + least + abs(c.scale) * P * ((dP - D).abs() * r + (3 * HS + 24) * U * (dPa + Da) + HS * 2.0 ** -29 * top(g)[:, None] * top(v)[None])
            nq = q.shape[0] * G
            for name, rows, X, eX, y in (("dq", (rq, h), dS, eS, k), ("dk", (rk, h // G), dS.T, eS.T, q),
                                         ("dv", (rk, h // G), P.T, (P * r + least).T, g)):
                terms = (2 * (n if name == "dq" else nq) + 32) * U
                size = X.abs() * top(y)[None]
                w[name][0][rows] += X @ y
                w[name][1][rows] += (eX + X.abs() * terms) @ y.abs() + size.sum(1, keepdim=True) * 2.0 ** -30 + \
                    (n if name == "dq" else nq) * 2.0 ** -28 * (size.amax(1, keepdim=True) if size.shape[1] else 0.0)
    return w


def check_forward(c):
    out, lse = c.forward()
    w = results(c)
    inside(out, *w["out"], "out")
    inside(lse, *w["lse"], "lse")


def check_backward(c):
    """Of the rounded results, which the kernels get as well."""
    out, lse = c.forward()
    w = results(c, lse, out)
    g = c.grads(3.0)
    c.backward(out, lse, g, zeroed=True)
    for name, x in zip(("dq", "dk", "dv"), g):
        inside(x, *w[name], name)


# (query lengths, key lengths, NH, NKV, HS): tiles of 64 and 32 keys, ragged heads, groups, a split key axis, few rows
SHAPES = [([40], [512], 2, 2, 64), ([300], None, 1, 1, 64), ([40], [512], 2, 1, 128), ([70, 33], None, 4, 1, 50), ([12], [3000], 2, 2, 64),
          ([130], None, 2, 2, 100), ([1, 3], [512, 70], 2, 2, 64), ([50], [200], 3, 3, 4)]


def large_value(gpu, size, lq, lk, NH, NKV, HS):
    """Key 5 has a weight near e^-80 or less in every row, and a value `size` times the others."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    c.q[:, :, 0] = 80.0 ** 0.5 / c.scale ** 0.5
    for k0 in c.s.k:
        c.k[k0 + 5, :, 0] = -(80.0 ** 0.5) / c.scale ** 0.5
        c.v[k0 + 5] *= size
    return c


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("size", [2.0 ** 12, 1e6, 1e10, 1e20])
def test_a_large_value_of_little_weight(gpu, size, lq, lk, NH, NKV, HS):
    check_forward(large_value(gpu, size, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("size", [2.0 ** 12, 1e6, 1e10])
def test_gradients_beside_a_large_value_of_little_weight(gpu, size, lq, lk, NH, NKV, HS):
    check_backward(large_value(gpu, size, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("first", [0, 5, 200])
def test_a_large_value_of_little_weight_two_blocks_a_wavefront(gpu, first):
    """As above where the call has so many rows that a wavefront takes two blocks of them."""
    c = Call(gpu, Seqs([40], [300]), 768, 768, 64)
    c.q[:, :, 0] = 80.0 ** 0.5 / c.scale ** 0.5
    c.k[first, :, 0] = -(80.0 ** 0.5) / c.scale ** 0.5
    c.v[first] *= 1e9
    out, _ = c.forward()
    c.NH = c.NKV = 8
    c.q, c.k, c.v, c.dout = (t[:, :8] for t in (c.q, c.k, c.v, c.dout))
    inside(out[:, :8], *results(c)["out"], "out")


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
def test_a_large_key_that_is_not_chosen(gpu, lq, lk, NH, NKV, HS):
    """A key 1e12 times the others whose score is far below theirs."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    c.q[:, :, 0] = 4.0
    for k0 in c.s.k:
        c.k[k0 + 7] *= 2.0
        c.k[k0 + 7, :, 0] = -1e12
    check_forward(c)


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("bits", [16, 30, 45])
def test_gradients_of_keys_of_little_weight(gpu, bits, lq, lk, NH, NKV, HS):
    """One key takes nearly all the weight: the others weigh about 2^-bits in every row, and their dv and dk have
    as many digits as the first one's."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    x = (bits * math.log(2.0) / c.scale) ** 0.5
    c.q[:, :, 0] = x
    c.k[:, :, 0] = 0.0
    for k0 in c.s.k:
        c.k[k0, :, 0] = x
    check_backward(c)


def by_row(c, spread, seed, which):
    """Rows of the tensors named in `which` times 2^e, e drawn from [-spread, spread] for each row."""
    g = torch.Generator().manual_seed(seed)
    for name in which:
        t = getattr(c, name)
        t.copy_(torch.ldexp(t, torch.randint(-spread, spread + 1, (t.shape[0], 1, 1), generator=g).to(DEV)))


SPREADS = [(8, "q k"), (4, "v dout"), (8, "v dout"), (20, "v dout"), (45, "v"), (45, "dout"), (6, "k v dout")]


def spread_rows(gpu, spread, which, lq, lk, NH, NKV, HS):
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS, scale=HS ** -0.5 * (2.0 ** -spread if "k" in which else 1.0))
    by_row(c, spread, spread, which.split())
    return c


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("spread,which", SPREADS)
def test_sizes_that_change_from_row_to_row(gpu, spread, which, lq, lk, NH, NKV, HS):
    check_forward(spread_rows(gpu, spread, which, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("spread,which", SPREADS)
def test_gradients_where_sizes_change_from_row_to_row(gpu, spread, which, lq, lk, NH, NKV, HS):
    check_backward(spread_rows(gpu, spread, which, lq, lk, NH, NKV, HS))


def large_blocks(gpu, seed):
    """Blocks of keys whose values, and scores, grow, shrink or alternate by large factors: what the sums stand on moves."""
    c = Call(gpu, Seqs([37], [700]), 2, 1, 64)
    at = torch.arange(700, device=DEV) // 32
    e = ((at * 3) % 23 if seed == 0 else 40 - 2 * at if seed == 1 else 40 * (at % 2)).clamp(-60, 60)
    c.v.copy_(torch.ldexp(c.v, e[:, None, None]))
    c.q[:, :, 0] = 8.0
    c.k[:, :, 0] = (at * (1, 3, 0)[seed] - 20).float()[:, None]
    return c


@pytest.mark.parametrize("seed", range(3))
def test_largest_values_first_last_and_between(gpu, seed):
    check_forward(large_blocks(gpu, seed))


@pytest.mark.parametrize("seed", range(3))
def test_gradients_of_largest_values_first_last_and_between(gpu, seed):
    check_backward(large_blocks(gpu, seed))


def ends(gpu, sizes, scale, lq, lk, NH, NKV, HS):
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS, scale=HS ** -0.5 * 2.0 ** scale)
    for name, e in zip(("q", "k", "v", "dout"), sizes):
        t = getattr(c, name)
        t.mul_(2.0 ** e)
    return c


ENDS = [((0, 0, -105, 0), 0), ((-105, 105, 0, -90), 0), ((-90, 100, 0, 0), -10), ((10, 10, 60, 40), -20)]


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("sizes,scale", ENDS)
def test_the_ends_of_the_range(gpu, sizes, scale, lq, lk, NH, NKV, HS):
    """Results near the least and the largest numbers have their digits."""
    check_forward(ends(gpu, sizes, scale, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("sizes,scale", ENDS)
def test_gradients_at_the_ends_of_the_range(gpu, sizes, scale, lq, lk, NH, NKV, HS):
    check_backward(ends(gpu, sizes, scale, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
def test_keys_of_minus_infinity_in_the_backward(gpu, lq, lk, NH, NKV, HS):
    """Keys whose scores are -infinity for an infinite element weigh nothing in the gradients either: dq is that of
    the other keys, theirs are 0. A row without another key has gradients 0."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 0.1
    for k0, n in zip(c.s.k, c.s.lk):
        c.k[k0 + n // 4:k0 + n, :, 0] = -math.inf
    out, lse = c.forward()
    finite = c.k.clone()
    finite[c.k == -math.inf] = 0.0
    short = Call(gpu, c.s, NH, NKV, HS)  # the same with those keys at a finite score far below
    short.q, short.v, short.dout, short.k = c.q, c.v, c.dout, finite.clone()
    short.k[:, :, 0][c.k[:, :, 0] == -math.inf] = -1e6
    w = results(short, lse, out)
    g, start = c.grads(3.0), 3.0
    c.backward(out, lse, g, zeroed=True)
    gone = c.k[:, :, 0] == -math.inf
    # a row that sees finite keys: those of -infinity reach nothing; a row that sees none: zeros
    for name, x in zip(("dq", "dk", "dv"), g):
        want, tol = w[name]
        if name == "dq":
            empty = lse == -math.inf
            assert x[empty].eq(0).all()
            inside(x[~empty], want[~empty], tol[~empty], name)
        else:
            assert x[gone].eq(0).all(), name
            keep = ~gone
            inside(x[keep], want[keep], tol[keep], name)
    # every key of -infinity: no gradients at all
    c.k[:, :, 0] = -math.inf
    out, lse = c.forward()
    assert out.eq(0).all() and (lse == -math.inf).all()
    g = c.grads(start)
    c.backward(out, lse, g, zeroed=True)
    assert all(x.eq(0).all() for x in g)


def test_queries_of_minus_infinity_in_the_backward(gpu):
    """A query row whose own infinite element makes all its scores -infinity: its gradients are 0 and it adds nothing
    to those of the keys."""
    c = Call(gpu, Seqs([70]), 2, 1, 64)
    c.k[:, :, 0] = c.k[:, :, 0].abs() + 0.1
    w = None
    clean = Call(gpu, Seqs([70]), 2, 1, 64)
    clean.k[:, :, 0] = clean.k[:, :, 0].abs() + 0.1
    clean.dout[33] = 0.0
    out, lse = clean.forward()
    out[33] = 0.0
    w = results(clean, lse, out)
    c.q[33, :, 0] = -math.inf
    out, lse = c.forward()
    assert out[33].eq(0).all() and (lse[33] == -math.inf).all()
    g = c.grads(2.0)
    c.backward(out, lse, g, zeroed=True)
    assert g[0][33].eq(0).all()
    rows = torch.arange(70, device=DEV) != 33
    inside(g[0][rows], w["dq"][0][rows], w["dq"][1][rows], "dq")
    inside(g[1], *w["dk"], "dk")
    inside(g[2], *w["dv"], "dv")


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
def test_scores_that_overflow_to_minus_infinity(gpu, lq, lk, NH, NKV, HS):
    """Finite queries and keys whose every product is beyond the range: out 0, lse -infinity, gradients 0."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    c.q[:] = 2.0 ** 64
    c.k[:] = -(2.0 ** 64)
    out, lse = c.forward()
    assert out.eq(0).all() and (lse == -math.inf).all()
    g = c.grads(2.0)
    c.backward(out, lse, g, zeroed=True)
    assert all(x.eq(0).all() for x in g)
    # from some key on: the rows hold what the keys before them give
    n0 = min(c.s.lk) // 2
    c.q[:], c.k[:] = 2.0 ** 60, -(2.0 ** 66)
    for k0 in c.s.k:
        c.k[k0:k0 + n0] = rand(torch.Generator(device=DEV).manual_seed(5), n0, NKV, HS) * 2.0 ** -62
    out, lse = c.forward()
    c.k.clamp_(min=-(2.0 ** 20))  # in 64 bits: scores far below
    w = results(c)
    inside(out, *w["out"], "out")


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3e38])
def test_rows_of_queries_that_cannot_be_used(gpu, value):
    """Query and dout rows of NaN, infinities or the largest values: dk and dv of the keys that they do not see, and dq of the
    other rows, have every digit."""
    for HS, n, r in ((64, 150, 20), (128, 150, 40), (50, 300, 130)):
        c = Call(gpu, Seqs([n]), 2, 1, HS)
        out, lse = c.forward()
        clean = Call(gpu, Seqs([n]), 2, 1, HS)
        c.q[r], c.dout[r] = value, value
        g = c.grads(5.0)
        c.backward(out, lse, g, zeroed=True)
        want = results(clean, lse, out)
        keys = torch.arange(n, device=DEV) > r
        others = torch.arange(n, device=DEV) != r
        inside(g[0][others], want["dq"][0][others], want["dq"][1][others], "dq of the other rows")
        inside(g[1][keys], want["dk"][0][keys], want["dk"][1][keys], "dk of the keys that the row does not see")
        inside(g[2][keys], want["dv"][0][keys], want["dv"][1][keys], "dv of the keys that the row does not see")


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("masked", ["all", "late"])
def test_scores_of_the_lowest_value(gpu, masked, lq, lk, NH, NKV, HS):
    """Keys masked by scores of the type's lowest value: they weigh nothing beside others, and among themselves the same
    (what else a score holds is far below its last bit)."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS, scale=1.0)
    c.q[:, :, 0] = 1.0
    lowest = -3.4028234663852886e38
    for k0, n in zip(c.s.k, c.s.lk):
        c.k[k0 if masked == "all" else k0 + n // 2:k0 + n, :, 0] = lowest
    out, lse = c.forward()
    for b in range(len(c.s.lq)):
        for h in range(NH):
            rq, rk, q, k, v = att_ref._pieces(c.s, b, h, NH // NKV, c.q, c.k, c.v)
            n = k.shape[0]
            ok = att_ref.allowed(q.shape[0], n, True, DEV)
            seen = ok.sum(1, keepdim=True)
            if masked == "all":
                # a mean of n values: n + 4 roundings of the sum of their sizes, the weights' 2^-22, and 2^-23 of the largest
                want, size = ok.double() @ v / seen, ok.double() @ v.abs() / seen
                inside(out[rq, h], want, size * (n + 64) * U + 2.0 ** -22 * v.abs().amax(), "out")
                assert (lse[rq, h] == lowest).all()
            else:
                few = ok[:, :n // 2]
                S = (q @ k[:n // 2].T).masked_fill(~few, -math.inf)
                es = (3 * HS + 16) * U * (q.abs() @ k[:n // 2].abs().T) + HS * 2.0 ** -29 * top(q)[:, None] * top(k[:n // 2])[None]
                P = torch.softmax(S, 1)
                rel = 2 * es.amax(1, keepdim=True) + 16 * U * (S.masked_fill(~few, 0.0).abs().amax(1, keepdim=True) + 4)
                want, size = P @ v[:n // 2], P @ v[:n // 2].abs()
                # e^x - 1 for the relative error x of a weight, which may pass 1 where scores are in the hundreds
                tol = size * (torch.expm1(rel) + (2 * n + 32) * U) + n * 2.0 ** -23 * (P * top(v[:n // 2])[None]).amax(1, keepdim=True)
                inside(out[rq, h], want, tol + 2.0 ** -29 * v.abs().amax(), "out")


def zero_rows(gpu, name, lq, lk, NH, NKV, HS):
    """Rows of zeros among the others, scores of up to hundreds: often all the weight falls on a value of zeros."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    by_row(c, 3, 11, ["q", "k"])
    t = getattr(c, name)
    t[torch.rand(t.shape[0], generator=torch.Generator().manual_seed(5)).to(DEV) < 0.3] = 0.0
    return c


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("name", ["k", "v"])
def test_rows_of_zeros(gpu, name, lq, lk, NH, NKV, HS):
    check_forward(zero_rows(gpu, name, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
def test_gradients_of_rows_of_zeros(gpu, name, lq, lk, NH, NKV, HS):
    check_backward(zero_rows(gpu, name, lq, lk, NH, NKV, HS))


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
@pytest.mark.parametrize("far", [30.0, 1000.0])
def test_all_the_weight_on_a_value_of_zeros(gpu, far, lq, lk, NH, NKV, HS):
    """The first key has a score `far` above the others and a value of zeros: what is left is the others', e^-far of them."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS)
    c.q[:, :, 0] = (far / c.scale) ** 0.5
    c.k[:, :, 0] = 0.0
    for k0 in c.s.k:
        c.k[k0, :, 0] = (far / c.scale) ** 0.5
        c.v[k0] = 0.0
    check_forward(c)
    check_backward(c)


@pytest.mark.parametrize("which,spread", [("k", 3), ("v", 12), ("zeros", 0)])
def test_sizes_that_change_with_two_blocks_a_wavefront(gpu, which, spread):
    """Keys and values of different sizes, and of zeros, where a wavefront takes two blocks of rows."""
    c = Call(gpu, Seqs([70], [300]), 800, 800, 64)
    if which == "zeros":
        c.v[::3] = 0.0
        c.q.mul_(8.0)
    else:
        by_row(c, spread, 3, [which])
    out, lse = c.forward()
    for heads in (slice(0, 3), slice(797, 800)):
        d = Call(gpu, c.s, 3, 3, 64)
        d.q, d.k, d.v = c.q[:, heads], c.k[:, heads], c.v[:, heads]
        w = results(d)
        inside(out[:, heads], *w["out"], "out")
        inside(lse[:, heads], *w["lse"], "lse")


@pytest.mark.parametrize("lq,lk,NH,NKV,HS", SHAPES)
def test_scores_near_the_highest_value(gpu, lq, lk, NH, NKV, HS):
    """One key at the highest score that is a number takes all the weight, NaN elsewhere stays NaN."""
    c = Call(gpu, Seqs(lq, lk), NH, NKV, HS, scale=1.0)
    c.q[:, :, 0] = 1.0
    for k0 in c.s.k:
        c.k[k0, :, 0] = 3.4028234663852886e38
    out, lse = c.forward()
    for b in range(len(c.s.lq)):
        for h in range(NH):
            rq, rk, q, k, v = att_ref._pieces(c.s, b, h, NH // NKV, c.q, c.k, c.v)
            assert (out[rq, h].double() - v[0]).abs().max() <= 2.0 ** -22 * v[0].abs().max()
            assert (lse[rq, h] == 3.4028234663852886e38).all()
    c.k[c.s.k[0], :, 0] = math.nan
    out, lse = c.forward()
    assert out[c.s.q[0]:c.s.q[0] + c.s.lq[0]].isnan().all()
