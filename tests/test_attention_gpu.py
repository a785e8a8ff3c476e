"""GPU: attention forward and backward against 64 bits at the lengths, heads, strides and masks where it can go
wrong, its refusals of bad offsets, graphs, streams, and a run of it inside the step driver."""
import math

import pytest
import torch

import att_ref
from att_ref import Seqs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Call:
    """Inputs of one call: q, k, v as views (rows, heads, HS) into buffers with `pad` floats between rows, the first
    element `off` floats into its buffer."""

    def __init__(self, gpu, s, NH, NKV, HS, causal=True, scale=None, pad=0, off=0, seed=1, sizes=(1.0, 1.0, 1.0), packed=False):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.gpu, self.s, self.causal = gpu, s, causal
        self.scale = HS ** -0.5 if scale is None else scale
        self.NH, self.NKV, self.HS = NH, NKV, HS
        if packed:  # q, k and v side by side, as the step driver's buffers hold them
            self.ldq = self.ldk = self.ldv = (NH + 2 * NKV) * HS + pad
            buf = rand(g, off + s.rows_q * self.ldq)
            self.q = self.view(buf[off:], s.rows_q, NH, self.ldq)
            self.k = self.view(buf[off + NH * HS:], s.rows_k, NKV, self.ldk)
            self.v = self.view(buf[off + (NH + NKV) * HS:], s.rows_k, NKV, self.ldv)
        else:
            self.ldq, self.ldk, self.ldv = NH * HS + pad, NKV * HS + pad, NKV * HS + 2 * pad
            mk = lambda rows, n, ld, z: self.view(rand(g, off + rows * ld + pad, scale=z)[off:], rows, n, ld)  # noqa: E731
            self.q = mk(s.rows_q, NH, self.ldq, sizes[0])
            self.k = mk(s.rows_k, NKV, self.ldk, sizes[1])
            self.v = mk(s.rows_k, NKV, self.ldv, sizes[2])
        self.ldo = NH * HS + pad
        self.dout = self.view(rand(g, off + s.rows_q * self.ldo)[off:], s.rows_q, NH, self.ldo)
        self.off = off

    def view(self, buf, rows, heads, ld):
        return buf.as_strided((rows, heads, self.HS), (ld, self.HS, 1), buf.storage_offset())

    def att(self, offsets=True):
        s = self.s
        o = {}
        if offsets:
            o = {"q_start": ints(s.q), "q_end": ints([a + n for a, n in zip(s.q, s.lq)]), "k_start": ints(s.k),
                 "k_end": ints([a + n for a, n in zip(s.k, s.lk)])}
        return self.gpu.Attention(nseq=len(s.lq), NH=self.NH, NKV=self.NKV, HS=self.HS, rows_q=s.rows_q, rows_k=s.rows_k,
                                  max_q=max(s.lq, default=0), max_k=max(s.lk, default=0), causal=self.causal, scale=self.scale,
                                  ldq=self.ldq, ldk=self.ldk, ldv=self.ldv, ldo=self.ldo, **o)

    def forward(self, offsets=True, lse=True):
        out = self.view(torch.full((self.off + self.s.rows_q * self.ldo,), 7.0, device=DEV)[self.off:], self.s.rows_q, self.NH, self.ldo)
        L = torch.full((self.s.rows_q, self.NH), 7.0, device=DEV)
        self.gpu.attention_forward(out, L if lse else None, self.q, self.k, self.v, self.att(offsets))
        return out, L

    def grads(self, value=0.0):
        mk = lambda rows, n, ld: self.view(torch.full((self.off + rows * ld,), value, device=DEV)[self.off:], rows, n, ld)  # noqa: E731
        return [mk(self.s.rows_q, self.NH, self.ldq), mk(self.s.rows_k, self.NKV, self.ldk), mk(self.s.rows_k, self.NKV, self.ldv)]

    def backward(self, out, lse, grads, zeroed=False):
        fn = self.gpu.attention_backward_zeroed if zeroed else self.gpu.attention_backward
        fn(*grads, self.dout, self.q, self.k, self.v, out, lse, self.att())


def inside(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & ~(got.double() == want)  # infinities equal
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol.clamp(min=1e-300))[bad].nan_to_num(1e9).max()):.3g} of the bound"


def rows_of(starts, lens, n):
    m = torch.zeros(n, dtype=torch.bool, device=DEV)
    for a, b in zip(starts, lens):
        m[a:a + b] = True
    return m


def check_forward(c, out, lse):
    w, wl, tol, tol_l = att_ref.forward(c.s, c.q, c.k, c.v, c.scale, c.causal)
    m = rows_of(c.s.q, c.s.lq, c.s.rows_q)
    inside(out[m], w[m], tol[m], "out")
    inside(lse[m], wl[m], tol_l[m], "lse")
    assert (out[~m] == 7.0).all() and (lse[~m] == 7.0).all(), "rows outside the sequences were written"


def check_backward(c, out, lse):
    """Both forms: added onto what the gradients hold, and written over it."""
    want, tol = att_ref.backward(c.s, c.q, c.k, c.v, out, lse, c.dout, c.scale, c.causal)
    mq, mk = rows_of(c.s.q, c.s.lq, c.s.rows_q), rows_of(c.s.k, c.s.lk, c.s.rows_k)
    for zeroed, start in ((False, 0.5), (True, 9.0)):
        g = c.grads(start)
        c.backward(out, lse, g, zeroed)
        for name, x, w, t, m in zip(("dq", "dk", "dv"), g, want, tol, (mq, mk, mk)):
            base = 0.0 if zeroed else start
            inside(x[m], w[m] + base, t[m] + 2.0 ** -24 * (w[m].abs() + t[m] + base), f"{name} zeroed={zeroed}")
            assert (x[~m] == start).all(), f"{name}: rows outside the sequences were written"


LENGTHS = {
    "one": ([1], None), "two": ([2, 1], None), "short": ([5, 0, 17, 1, 31, 32, 33], None),
    "tile": ([63, 64, 65], None), "edge": ([127, 128, 129], None), "long": ([300, 257, 1], None),
    "chunk": ([3, 16, 40], [50, 16, 333]), "token": ([1, 1, 1, 1], [1, 700, 64, 129]), "few": ([2, 4, 3], [300, 5, 1030]),
    "later": ([20, 70, 5], [7, 64, 0]),  # more query rows than keys: the first rows see nothing
    "nokeys": ([3, 1], [0, 0]), "noqueries": ([0, 0], [5, 40]),
}


@pytest.mark.parametrize("NH,NKV,HS", [(1, 1, 64), (6, 2, 64), (3, 3, 128), (8, 1, 16), (4, 4, 50), (5, 1, 33), (2, 2, 1), (2, 1, 80)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_forward_and_backward(gpu, lens, NH, NKV, HS):
    s = Seqs(*LENGTHS[lens], gap=1, tail=3)
    c = Call(gpu, s, NH, NKV, HS)
    out, lse = c.forward()
    check_forward(c, out, lse)
    check_backward(c, out, lse)


@pytest.mark.parametrize("NH,NKV,HS,pad,off", [(2, 2, 64, 0, 1), (4, 2, 64, 3, 2), (3, 1, 96, 5, 3), (2, 2, 128, 4, 4), (2, 2, 7, 1, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_strides_alignment_and_no_causal_limit(gpu, causal, NH, NKV, HS, pad, off):
    for lens, lk in (([70, 130], None), ([9, 33], [100, 20]), ([1, 2], [90, 300])):
        c = Call(gpu, Seqs(lens, lk, gap=2, tail=1), NH, NKV, HS, causal, pad=pad, off=off, packed=lk is None)
        out, lse = c.forward()
        check_forward(c, out, lse)
        check_backward(c, out, lse)


@pytest.mark.parametrize("B,T,NH", [(4, 64, 6), (2, 100, 3), (3, 1, 2)])
def test_equal_lengths_without_offsets(gpu, B, T, NH):
    c = Call(gpu, Seqs([T] * B), NH, NH, 64, packed=True)
    out, lse = c.forward(offsets=False)
    again, _ = c.forward(offsets=True, lse=False)
    assert torch.equal(out, again)
    check_forward(c, out, lse)


@pytest.mark.parametrize("sizes,scale", [((30.0, 30.0, 1.0), None), ((1e-6, 1e-4, 1e-3), None), ((1e-6, 1e6, 1e6), None),
                                         ((1e10, 1e-10, 1e20), None), ((1e-15, 1e15, 1e-25), None), ((1.0, 1.0, 1.0), 0.0),
                                         ((1.0, 1.0, 1.0), -3.0)])
def test_sizes_of_values(gpu, sizes, scale):
    """Values far from 1, scores up to thousands (one key takes all), equal scores, a negative scale."""
    for lens, lk in (([130, 65], None), ([1], [200])):
        c = Call(gpu, Seqs(lens, lk), 2, 1, 64, scale=scale, sizes=sizes)
        out, lse = c.forward()
        check_forward(c, out, lse)
        if max(sizes) <= 1e6 and min(sizes) >= 1e-6:
            check_backward(c, out, lse)


def test_one_row_of_outliers(gpu):
    """One key and one value a million times the others': what lies below them keeps its digits."""
    c = Call(gpu, Seqs([150]), 2, 2, 64)
    c.k[70] *= 1e4
    c.v[90] *= 1e6
    out, lse = c.forward()
    check_forward(c, out, lse)
    check_backward(c, out, lse)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, -3.4028234663852886e38])
def test_what_a_row_must_not_see_does_not_reach_it(gpu, value):
    """Unusable values behind the sequences, between them, and in the rows that come later than a row."""
    for lens, lk, NH, NKV, HS in (([100, 37], None, 2, 1, 64), ([9, 1], [70, 90], 2, 2, 64), ([64, 64], None, 1, 1, 128), ([40], None, 2, 2, 50)):
        s = Seqs(lens, lk, gap=2, tail=5)
        c = Call(gpu, s, NH, NKV, HS)
        out0, lse0 = c.forward()
        g0 = c.grads()
        c.backward(out0, lse0, g0)
        mq, mk = rows_of(s.q, s.lq, s.rows_q), rows_of(s.k, s.lk, s.rows_k)
        for t, m in ((c.q, mq), (c.k, mk), (c.v, mk), (c.dout, mq)):
            t[~m] = value
        out, lse = c.forward()
        assert torch.equal(out, out0) and torch.equal(lse, lse0)
        g = c.grads()
        c.backward(out, lse, g)
        for x, y in zip(g, g0):
            assert torch.equal(x, y)
        # the last key of each sequence: only the last query row sees it (bounds of 64 bits without it)
        last_k = [a + n - 1 for a, n in zip(s.k, s.lk) if n]
        last_q = [a + n - 1 for a, n in zip(s.q, s.lq) if n]
        w, wl, tol, tol_l = att_ref.forward(s, c.q, c.k, c.v, c.scale, True)
        c.k[last_k] = value
        c.v[last_k] = value
        out, lse = c.forward()
        m = mq.clone()
        m[last_q] = False
        inside(out[m], w[m], tol[m], "out of the rows before the last")
        inside(lse[m], wl[m], tol_l[m], "lse of the rows before the last")


def test_values_that_cannot_be_used_in_the_backward(gpu):
    """NaN in the last query row's q and dout and in the last key: gradients of what does not meet them are finite and
    equal to 64 bits."""
    s = Seqs([100])
    c = Call(gpu, s, 1, 1, 64)
    out, lse = c.forward()
    c.k[99], c.v[99] = math.nan, math.nan
    c2 = Call(gpu, Seqs([99], tail=1), 1, 1, 64)  # the same inputs without the last row
    assert torch.equal(c.q, c2.q)
    g = c.grads()
    c.backward(out, lse, g)
    want, tol = att_ref.backward(c2.s, c2.q, c2.k, c2.v, out, lse, c2.dout, c.scale, True)
    inside(g[0][:99], want[0][:99], tol[0][:99], "dq")


def test_infinite_values_that_a_row_sees(gpu):
    """An infinite value with weight: the output of the rows that see it is that infinity, as in any arithmetic."""
    c = Call(gpu, Seqs([80]), 1, 1, 64)
    c.v[20, 0, 3] = math.inf
    c.v[20, 0, 4] = -math.inf
    out, lse = c.forward()
    assert (out[20:, 0, 3] == math.inf).all() and (out[20:, 0, 4] == -math.inf).all()
    assert out[:20].isfinite().all() and out[:, 0, 5:].isfinite().all() and lse.isfinite().all()
    c.k[30, 0, 0] = math.nan
    out, lse = c.forward()
    assert out[30:].isnan().all() and lse[30:].isnan().all() and lse[:30].isfinite().all()


@pytest.mark.parametrize("lens,lk,NH,NKV,HS", [([700, 900], None, 12, 12, 64), ([1025, 3, 500], None, 8, 2, 128),
                                               ([1] * 6, [4000, 1, 513, 2222, 63, 64], 8, 2, 64), ([64], [3001], 4, 4, 64)])
def test_larger(gpu, lens, lk, NH, NKV, HS):
    c = Call(gpu, Seqs(lens, lk), NH, NKV, HS, packed=lk is None)
    out, lse = c.forward()
    check_forward(c, out, lse)
    check_backward(c, out, lse)
    again, lse2 = c.forward()
    assert torch.equal(out, again) and torch.equal(lse, lse2), "two calls differ"
    g1, g2 = c.grads(), c.grads()
    c.backward(out, lse, g1)
    c.backward(out, lse, g2)
    assert all(torch.equal(a, b) for a, b in zip(g1, g2)), "two backward calls differ"


def test_shared_prefix_rows_in_the_forward(gpu):
    """Sequences may share key rows."""
    c = Call(gpu, Seqs([1, 1, 2], [80, 80, 80]), 4, 2, 64)
    s = c.s
    s.k = [0, 0, 10]
    out, lse = c.forward()
    check_forward(c, out, lse)


def test_gradient_against_differences(gpu):
    """The directional derivative of sum(out * dout), by central differences in 64 bits: off by h^2 / 6 of its third
    derivative (for h = 1e-4 and values of order 1 below 1e-6 of the sum of the terms' sizes) and by the gradient's bound."""
    c = Call(gpu, Seqs([40, 9], [40, 30]), 4, 2, 64)
    out, lse = c.forward()
    g = c.grads()
    c.backward(out, lse, g)
    _, tol = att_ref.backward(c.s, c.q, c.k, c.v, out, lse, c.dout, c.scale, True)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(9)
    for which in range(3):
        d = torch.randn(g[which].shape, generator=gen, device=DEV, dtype=torch.float64)
        h, f = 1e-4, []
        for sign in (1, -1):
            t = [x.double() for x in (c.q, c.k, c.v)]
            t[which] = t[which] + sign * h * d
            f.append(float((att_ref.forward(c.s, *t, c.scale, True)[0] * c.dout.double()).sum()))
        got = float((g[which].double() * d).sum())
        bound = float((tol[which] * d.abs()).sum()) + 1e-6 * float((g[which].double().abs() * d.abs()).sum())
        assert abs(got - (f[0] - f[1]) / (2 * h)) <= bound


@pytest.mark.parametrize("bad", ["start", "end", "order", "long"])
def test_bad_offsets_are_clamped_and_reported(gpu, bad):
    c = Call(gpu, Seqs([20, 30], tail=2), 2, 2, 64)
    a = c.att()
    t = {"start": a._tensors[0], "end": a._tensors[3], "order": a._tensors[1], "long": a._tensors[1]}[bad]
    t[0] = {"start": -5, "end": 1000, "order": -7, "long": 45}[bad]
    out, lse = torch.zeros(52, 2, 64, device=DEV), torch.zeros(52, 2, device=DEV)
    gpu.attention_forward(out, lse, c.q, c.k, c.v, a)
    with pytest.raises(gpu.UgkError, match="attention_forward"):
        gpu.synchronize()
    g = c.grads()
    gpu.attention_backward(*g, c.dout, c.q, c.k, c.v, out, lse, a)
    with pytest.raises(gpu.UgkError, match="attention_backward"):
        gpu.synchronize()
    gpu.synchronize()  # the report is cleared
    assert out[50:].eq(0).all()


@pytest.mark.parametrize("lens,lk", [([100, 60], None), ([1, 1], [700, 90])])
def test_captured_and_replayed(gpu, lens, lk):
    """A captured forward and backward replayed with eager calls of another shape between, each replay checked."""
    c, other = Call(gpu, Seqs(lens, lk), 4, 2, 64), Call(gpu, Seqs([33, 80]), 2, 2, 64, seed=5)
    a, oa = c.att(), other.att()
    out, lse = c.forward()
    g = c.grads()
    c.backward(out, lse, g)
    want = [t.clone() for t in (out, lse, *g)]
    o_out, o_lse = other.forward()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for t in g:
                t.zero_()
            gpu.attention_forward(out, lse, c.q, c.k, c.v, a)
            gpu.attention_backward(*g, c.dout, c.q, c.k, c.v, out, lse, a)
        for _ in range(3):
            for t in (out, lse, *g):
                t.fill_(3.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for x, w in zip((out, lse, *g), want):
                assert torch.equal(x, w)
            x, y = torch.empty_like(o_out), torch.empty_like(o_lse)
            with torch.cuda.stream(stream):
                gpu.attention_forward(x, y, other.q, other.k, other.v, oa)
                gpu.attention_backward(*other.grads(), other.dout, other.q, other.k, other.v, x, y, oa)
            stream.synchronize()
            assert torch.equal(x, o_out) and torch.equal(y, o_lse)
    finally:
        gpu.set_stream(None)


def test_dense_callbacks_in_the_step_driver(gpu):
    """The step driver with the library's attention and torch's products: the attention buffers of every block hold
    what 64 bits give for the block's qkv, and the gradients accumulate onto the callback's dqkv."""
    cfg = gpu.Config(B=3, T=40, C=128, V=50, NH=2, maxT=64, L=2)
    B, T, C, NH = cfg.B, cfg.T, cfg.C, cfg.NH
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    qkv = rand(g, B * T, 3 * C)
    dout, base = rand(g, B * T, C), rand(g, B * T, 3 * C)
    s = Seqs([T] * B)
    q, k, v = (qkv[:, i * C:(i + 1) * C].unflatten(1, (NH, C // NH)) for i in range(3))
    w, wl, tol, _ = att_ref.forward(s, q, k, v, (C // NH) ** -0.5, True)
    out = torch.empty(B * T, C, device=DEV)
    gpu.dense_attention_forward(out, qkv, B, T, C, NH)
    inside(out.view(B * T, NH, -1), w, tol, "dense forward")
    dqkv = base.clone()
    gpu.dense_attention_backward(dqkv, dout, qkv, B, T, C, NH)
    # the callback's own out and lse are within tol of these, which moves D by at most sum |dout| tol
    grads, gt = att_ref.backward(s, q, k, v, w.float(), wl.float(), dout.unflatten(1, (NH, C // NH)), (C // NH) ** -0.5, True)
    for i, (x, t) in enumerate(zip(grads, gt)):
        got = (dqkv - base)[:, i * C:(i + 1) * C].unflatten(1, (NH, C // NH))
        inside(got, x, 4 * t + 2.0 ** -23 * base[:, i * C:(i + 1) * C].unflatten(1, (NH, C // NH)).abs() + 2.0 ** -23, f"dense gradient {i}")
    # inside the driver: the qkv buffers as they are (no products), attention by the library
    params = rand(g, gpu.param_count(cfg), scale=0.02)
    acts = rand(g, gpu.act_count(cfg))
    inp = torch.randint(0, cfg.V, (B * T,), generator=g, device=DEV, dtype=torch.int32)
    ops = gpu.DenseOps(**gpu.dense_attention_callbacks())
    n = B * T * C
    block = 18 * n + 4 * B * T
    gpu.gpt2_layers_forward(acts, params, inp, cfg, ops)
    for l in range(cfg.L):
        at = n + l * block + n + 2 * B * T
        blk_qkv, atty = acts[at:at + 3 * n].view(B * T, 3 * C), acts[at + 3 * n:at + 4 * n]
        gpu.dense_attention_forward(out, blk_qkv.contiguous(), B, T, C, NH)
        assert torch.equal(atty, out.view(-1)), f"block {l}"
    grads, ga = torch.zeros(gpu.param_count(cfg), device=DEV), torch.zeros(gpu.act_count(cfg), device=DEV)
    ga[n + cfg.L * block:n + cfg.L * block + n] = rand(g, n)
    for l in range(cfg.L):
        at = n + l * block + n + 2 * B * T
        ga[at + 3 * n:at + 4 * n] = rand(g, n)
    gpu.gpt2_layers_backward(grads, ga, acts, params, inp, cfg, ops)
    for l in range(cfg.L):
        at = n + l * block + n + 2 * B * T
        want = torch.zeros(3 * n, device=DEV)
        gpu.dense_attention_backward(want, ga[at + 3 * n:at + 4 * n].clone(), acts[at:at + 3 * n].clone(), B, T, C, NH)
        assert torch.equal(ga[at:at + 3 * n], want), f"gradient of block {l}"
    gpu.synchronize()


def test_caller_owned_workspace(gpu):
    """Inside a workspace sized for the config, and refused by one too small."""
    cfg = gpu.Config(B=2, T=64, C=128, V=50, NH=2, maxT=64, L=1)
    c, big = Call(gpu, Seqs([64, 64]), 2, 2, 64, packed=True), Call(gpu, Seqs([1] * 4000), 64, 64, 4)
    out, lse = c.forward()
    g = c.grads()
    c.backward(out, lse, g)
    b_out, b_lse = big.forward()
    n = gpu.workspace_bytes(cfg)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=DEV)
    at = (-ws.data_ptr()) % 256
    try:
        gpu.set_workspace(ws[at:at + n], cfg)
        out2, lse2 = c.forward()
        g2 = c.grads()
        c.backward(out2, lse2, g2)
        assert torch.equal(out, out2) and all(torch.equal(x, y) for x, y in zip(g, g2))
        rows = attention_rows_beyond(gpu, cfg, n)
        huge = Call(gpu, Seqs([1] * rows), 64, 64, 1)
        h_out, h_lse = torch.zeros(rows, 64, device=DEV), torch.zeros(rows, 64, device=DEV)
        with pytest.raises(gpu.UgkError) as err:
            huge.backward(h_out, h_lse, huge.grads())
        assert err.value.status == 3 and "attention" in str(err.value)
    finally:
        gpu.set_workspace(None, cfg)


def attention_rows_beyond(gpu, cfg, n):
    """Rows whose 64 row sums each exceed any region of a workspace of n bytes."""
    return n // 256 + 1


def own_size_bounds(s, q, k, v, out, lse, dout, scale):
    """Bounds for one causal sequence from the sizes of what a row sees alone. An element is held to 2^-24 of itself
    and 2^-27 of the largest of its own row (a tile that not all rows see holds no row more than 2^13 below its
    largest) or 2^-40 of the largest that the row sees; the weights and dS to 2^-33 of the largest that it has seen."""
    n, HS = q.shape[0], q.shape[2]
    Q, K, V, O, G = (t[:, 0].double() for t in (q, k, v, out, dout))
    ok = att_ref.allowed(n, n, True, DEV)
    top = lambda t: t.abs().amax(1)  # noqa: E731
    es = abs(scale) * (HS + 8) * 2.0 ** -23 * HS * top(Q)[:, None] * top(K)[None]
    S = (Q @ K.T * scale).masked_fill(~ok, -math.inf)
    P = torch.exp(S - lse.double())
    rel = torch.where(ok, 2 * es + (S - lse.double()).abs().clamp(0, 90) * 2.0 ** -24, 0.0).amax(1, keepdim=True) * 2 + (2 * n + 32) * 2.0 ** -24
    floor = n * 2.0 ** -33
    seen_v = torch.cummax(top(V), 0).values
    t_out = (P * rel) @ top(V)[:, None] + floor * seen_v[:, None]
    D = (G.abs() * O.abs()).sum(1)
    size = torch.where(ok, P * abs(scale) * (HS * top(G)[:, None] * top(V)[None] + D[:, None]), 0.0)
    more = rel + (2 * HS + 32) * 2.0 ** -24
    seen_k = torch.cummax(top(K), 0).values
    worst = size.amax(1)
    t_q = (size * more) @ top(K)[:, None] + floor * (worst * seen_k)[:, None]
    back = lambda t: torch.cummax(t.flip(0), 0).values.flip(0)  # noqa: E731
    t_k = (size * more).T @ top(Q)[:, None] + floor * (size.amax(0) * back(top(Q)))[:, None]
    t_v = (P * more).T @ top(G)[:, None] + floor * back(top(G))[:, None]
    return t_out, (t_q, t_k, t_v)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("n", [65, 129, 300])
def test_sizes_that_change_along_the_sequence(gpu, n, seed):
    """Values and gradients whose size jumps by up to 2^40 from one block of rows to the next, or in the last row
    alone: what a row does not see costs it no digits."""
    c = Call(gpu, Seqs([n]), 1, 1, 64, seed=seed)
    g = torch.Generator().manual_seed(seed)
    step = (32, 64, n - 1, 7)[seed]
    e = torch.randint(-20, 21, (n // step + 1,), generator=g).repeat_interleave(step)[:n].to(DEV)
    e2 = torch.randint(-20, 21, (n // step + 1,), generator=g).repeat_interleave(step)[:n].to(DEV)
    if seed == 2:
        e[:], e2[:] = 0, 0
        e[-1], e2[0] = 100, 60
    c.v.copy_(torch.ldexp(c.v, e[:, None, None]))
    c.dout.copy_(torch.ldexp(c.dout, e2[:, None, None]))
    out, lse = c.forward()
    w, wl, _, tol_l = att_ref.forward(c.s, c.q, c.k, c.v, c.scale, True)
    t_out, tols = own_size_bounds(c.s, c.q, c.k, c.v, w.float(), wl.float(), c.dout, c.scale)
    inside(out[:, 0], w[:, 0], t_out.expand(-1, 64), "out")
    inside(lse, wl, tol_l, "lse")
    gr = c.grads()
    c.backward(out, lse, gr, zeroed=True)
    want, _ = att_ref.backward(c.s, c.q, c.k, c.v, out, lse, c.dout, c.scale, True)
    for name, x, y, t in zip(("dq", "dk", "dv"), gr, want, tols):
        inside(x[:, 0], y[:, 0], t.expand(-1, 64), name)


@pytest.mark.parametrize("n", [65, 130])
def test_keys_whose_size_changes_along_the_sequence(gpu, n):
    """Keys and queries whose size jumps, the scores staying of order one to a thousand."""
    c = Call(gpu, Seqs([n]), 1, 1, 64)
    e = (torch.arange(n, device=DEV) // 32 % 2) * 10
    c.k.copy_(torch.ldexp(c.k, -e[:, None, None]))
    c.q.copy_(torch.ldexp(c.q, (3 - e)[:, None, None]))
    c.k[-1] *= 2.0 ** 20
    c.q[0] *= 2.0 ** 15
    out, lse = c.forward()
    w, wl, _, _ = att_ref.forward(c.s, c.q, c.k, c.v, c.scale, True)
    t_out, tols = own_size_bounds(c.s, c.q, c.k, c.v, w.float(), wl.float(), c.dout, c.scale)
    inside(out[:, 0], w[:, 0], t_out.expand(-1, 64), "out")
    gr = c.grads()
    c.backward(out, lse, gr, zeroed=True)
    want, _ = att_ref.backward(c.s, c.q, c.k, c.v, out, lse, c.dout, c.scale, True)
    for name, x, y, t in zip(("dq", "dk", "dv"), gr, want, tols):
        inside(x[:, 0], y[:, 0], t.expand(-1, 64), name)


@pytest.mark.parametrize("lens,lk", [([70], None), ([2], [300]), ([1], [4000]), ([40], [1000])])
def test_scores_of_minus_infinity(gpu, lens, lk):
    """Keys whose scores are -infinity weigh nothing; a row that sees no others has out 0, lse -infinity, gradients 0.
    The same in every kernel and in every part of a split key axis."""
    c = Call(gpu, Seqs(lens, lk), 2, 1, 64)
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 0.1
    nk = c.s.lk[0]
    gone = slice(nk // 4, nk)
    c.k[gone, :, 0] = -math.inf
    out, lse = c.forward()
    # the rows as if the sequence ended before those keys
    q, k, v = c.q.double(), c.k[:nk // 4].double(), c.v[:nk // 4].double()
    for h in range(2):
        z = q[:, h] @ k[:, 0].T * c.scale
        if lk is None:
            z = z.masked_fill(~att_ref.allowed(lens[0], nk, True, DEV)[:, :nk // 4], -math.inf)
        p = torch.softmax(z, 1)
        assert torch.allclose(out[:, h].double(), p @ v[:, 0], rtol=1e-4, atol=1e-5)
        assert torch.allclose(lse[:, h].double(), torch.logsumexp(z, 1), rtol=1e-5, atol=1e-5)
    g = c.grads()
    c.backward(out, lse, g)
    assert g[2][gone].eq(0).all()
    c.k[:, :, 0] = -math.inf
    out, lse = c.forward()
    assert out.eq(0).all() and (lse == -math.inf).all()
    g = c.grads()
    c.backward(out, lse, g)
    assert g[2].eq(0).all()


@pytest.mark.parametrize("Q", [1, 12])
def test_offsets_beyond_32_bits(gpu, Q):
    """A cache of more than 2^31 floats, the sequences at its end."""
    NH, HS, ld, n = 2, 64, 4096, 200
    rows = 2 ** 31 // ld + 600
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    k = torch.empty(rows * ld, device=DEV)
    starts = [rows - 500, rows - n]
    tail = k[(rows - 500) * ld:]
    tail.copy_(torch.randn(tail.numel(), generator=g, device=DEV))
    q = rand(g, 2 * Q, NH * HS)
    out, lse = torch.empty(2 * Q, NH * HS, device=DEV), torch.empty(2 * Q, NH, device=DEV)
    a = gpu.Attention(nseq=2, NH=NH, NKV=NH, HS=HS, rows_q=2 * Q, rows_k=rows, max_q=Q, max_k=n, q_start=ints([0, Q]),
                      q_end=ints([Q, 2 * Q]), k_start=ints(starts), k_end=ints([s + n for s in starts]), ldk=ld, ldv=ld)
    gpu.attention_forward(out, lse, q, k, k[NH * HS:], a)
    gpu.synchronize()
    t = tail.view(-1, ld)
    s = Seqs([Q, Q], [n, n])
    s.k, s.rows_k = [0, 500 - n], 500
    kk, vv = t[:, :NH * HS].unflatten(1, (NH, HS)), t[:, NH * HS:2 * NH * HS].unflatten(1, (NH, HS))
    w, wl, tol, tol_l = att_ref.forward(s, q.view(2 * Q, NH, HS), kk, vv, HS ** -0.5, True)
    inside(out.view(2 * Q, NH, HS), w, tol, "out")
    inside(lse, wl, tol_l, "lse")


def test_many_sequences(gpu):
    """More (sequence, head) pairs than a launch has XCDs, CUs or parts for, of every length from 0 to 40."""
    lens = [(7 * i) % 41 for i in range(700)]
    for lq, lk in ((lens, None), ([1] * 700, lens)):
        c = Call(gpu, Seqs(lq, lk), 2, 1, 8)
        out, lse = c.forward()
        check_forward(c, out, lse)
        check_backward(c, out, lse)


def test_backward_workspace_of_a_large_cache(gpu):
    """The parts of dk and dv hold all key rows: where the sequences are a small part of a cache, there are few."""
    n, rows_k, NH, HS = 1100, 1 << 20, 2, 64
    c = Call(gpu, Seqs([n], [n]), NH, 1, HS)
    c.s.k, c.s.rows_k = [rows_k - n], rows_k
    k, v = (torch.zeros(rows_k, 1, HS, device=DEV) for _ in range(2))
    k[-n:], v[-n:] = c.k, c.v
    c.k, c.v = k, v
    out, lse = c.forward()
    grads = c.grads()
    gpu.synchronize()
    free = torch.cuda.mem_get_info()[0]
    c.backward(out, lse, grads)
    gpu.synchronize()
    # the bound: 2 * 8 parts of 2^20 rows would be 4.3 GB
    assert free - torch.cuda.mem_get_info()[0] < 1 << 30
    s = Seqs([n], [n])
    want, tol = att_ref.backward(s, c.q, k[-n:], v[-n:], out, lse, c.dout, c.scale, True)
    for got, w, t, name in zip((grads[0], grads[1][-n:], grads[2][-n:]), want, tol, ("dq", "dk", "dv")):
        inside(got, w, t, name)
    assert not grads[1][:-n].any() and not grads[2][:-n].any()


@pytest.mark.parametrize("lens,lk", [([300, 41], None), ([1, 1], [700, 90]), ([2], [2000])])
def test_limits_far_above_the_buffers(gpu, lens, lk):
    """max_q and max_k of the longest sequence that there could be, not of this call's."""
    c = Call(gpu, Seqs(lens, lk), 4, 2, 64)
    out, lse = c.forward()
    a = c.att()
    a.max_q = a.max_k = 2 ** 31 - 1
    out2, lse2, grads2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0), c.grads()
    gpu.attention_forward(out2, lse2, c.q, c.k, c.v, a)
    gpu.attention_backward(*grads2, c.dout, c.q, c.k, c.v, out2, lse2, a)
    gpu.synchronize()
    check_forward(c, out2, lse2)
    want, tol = att_ref.backward(c.s, c.q, c.k, c.v, out2, lse2, c.dout, c.scale, True)
    for got, w, t, name in zip(grads2, want, tol, ("dq", "dk", "dv")):
        inside(got, w, t, name)


def test_tensors_that_the_binding_refuses(gpu, monkeypatch):
    """Offsets for fewer sequences than asked for, rows whose elements are apart, tensors on another GPU."""
    c = Call(gpu, Seqs([4, 3]), 2, 2, 64)
    out, lse = c.forward()
    a = c.att()
    a.nseq = 3
    with pytest.raises(ValueError, match="the offsets hold 2"):
        gpu.attention_forward(out, lse, c.q, c.k, c.v, a)
    with pytest.raises(ValueError, match="the offsets hold 2"):
        c.gpu.attention_backward(*c.grads(), c.dout, c.q, c.k, c.v, out, lse, a)
    wide = torch.zeros(128, 7, device=DEV).t()
    with pytest.raises(ValueError, match="last stride"):
        gpu.attention_forward(out, lse, wide, c.k, c.v, c.att())
    a, x = c.att(), torch.zeros(64, device=DEV)
    monkeypatch.setattr(gpu, "_one_device", False)
    assert torch.cuda.current_device() == 0
    gpu.attention_forward(out, lse, c.q, c.k, c.v, a)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: gpu.attention_forward(out, lse, c.q, c.k, c.v, a), lambda: gpu.dropout_forward(x, x, 64, 0.5, 1, 1),
                 lambda: gpu.attention_forward(1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, a),
                 lambda: gpu.attention_forward(1 << 20, lse, 1 << 20, 1 << 20, 1 << 20, gpu.Attention(1, 2, 2, 64, 7, 7, 7, 7)),
                 lambda: gpu.dense_attention_forward(x, torch.zeros(192, device=DEV), 1, 1, 64, 1)):
        with pytest.raises(ValueError, match="the current device is cuda:1"):
            call()


def test_a_graph_keeps_its_workspace_when_the_region_grows(gpu):
    """A captured call, then a call that needs a larger workspace, then other memory written: the replay's results stay."""
    cfg = gpu.Config(B=1, T=64, C=64, V=50, NH=1, maxT=64, L=1)
    ws = torch.empty(gpu.workspace_bytes(cfg) + 256, dtype=torch.uint8, device=DEV)
    at = (-ws.data_ptr()) % 256
    gpu.set_workspace(ws[at:at + gpu.workspace_bytes(cfg)], cfg)
    gpu.set_workspace(None, cfg)  # the library's own regions start again from nothing
    c, big = Call(gpu, Seqs([1, 1], [3000, 2500]), 2, 2, 64), Call(gpu, Seqs([3000]), 40, 40, 8)
    a = c.att()
    want, want_lse = c.forward()
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            gpu.attention_forward(out, lse, c.q, c.k, c.v, a)
        before = gpu.lib.ugk_scratch_bytes()
        with torch.cuda.stream(stream):
            b_out, b_lse = big.forward()
            big.backward(b_out, b_lse, big.grads())
        stream.synchronize()
        assert gpu.lib.ugk_scratch_bytes() > before
        for _ in range(3):
            out.fill_(3.0)
            lse.fill_(3.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
    finally:
        gpu.set_stream(None)


def test_capture_without_the_workspace_is_refused(gpu):
    cfg = gpu.Config(B=1, T=64, C=64, V=50, NH=1, maxT=64, L=1)
    ws = torch.empty(gpu.workspace_bytes(cfg) + 256, dtype=torch.uint8, device=DEV)
    at = (-ws.data_ptr()) % 256
    gpu.set_workspace(ws[at:at + gpu.workspace_bytes(cfg)], cfg)
    gpu.set_workspace(None, cfg)
    c = Call(gpu, Seqs([1, 1], [3000, 2500]), 2, 2, 64)
    a, x, y = c.att(), torch.zeros(2, 2, 64, device=DEV), torch.zeros(2, 2, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(gpu.UgkError) as err:
                gpu.attention_forward(x, y, c.q, c.k, c.v, a)
        assert err.value.status == 3 and "before graph capture" in str(err.value)
    finally:
        gpu.set_stream(None)
    out, lse = c.forward()
    check_forward(c, out, lse)


@pytest.mark.parametrize("HS", [65, 68, 80, 96, 100, 124, 126, 127])
def test_head_sizes_above_64(gpu, HS):
    c = Call(gpu, Seqs([150, 3, 0, 70], gap=1, tail=2), 4, 2, HS, pad=3, off=1)
    out, lse = c.forward()
    check_forward(c, out, lse)
    check_backward(c, out, lse)


@pytest.mark.parametrize("NH,NKV,HS,Q,lens", [(16, 2, 128, 1, [5000, 1, 0, 1025]), (8, 8, 64, 8, [4100, 1024, 7]), (12, 2, 40, 9, [3001, 2047])])
def test_one_tile_of_rows_against_a_long_cache(gpu, NH, NKV, HS, Q, lens):
    c = Call(gpu, Seqs([Q] * len(lens), lens, gap=1), NH, NKV, HS)
    out, lse = c.forward()
    check_forward(c, out, lse)
    check_backward(c, out, lse)
