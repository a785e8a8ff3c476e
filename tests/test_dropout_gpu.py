"""GPU: dropout and its residual and LayerNorm pairs. The flat ops are single roundings of their formulas: bit for
bit. The pairs with LayerNorm give the bits of the ops that they name."""
import math

import numpy as np
import pytest
import torch

import drop_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SEED = 0x1234_5678_9ABC


def rand(n, seed, off=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(n + off, generator=g, device=DEV)[off:]


def same(got, want, what):
    got = got.cpu().numpy().view(np.uint32)
    want = np.ascontiguousarray(want, np.float32).view(np.uint32)
    assert np.array_equal(got, want), f"{what}: {(got != want).sum()} of {want.size} differ"


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 255, 1023, 2047, 2048, 2049, 2050, 4096, 98304, 300001])
@pytest.mark.parametrize("p,off", [(0.1, 0), (0.5, 1), (0.0, 2), (0.999, 3)])
def test_flat_ops(gpu, n, p, off):
    x, y, a, b = (rand(n, k, off) for k in range(4))
    h = [t.cpu().numpy() for t in (x, y, a, b)]
    kept = drop_ref.keep(n, p, SEED, 5, 2)
    drop = lambda v: drop_ref.drop(v, kept, p)  # noqa: E731
    out = torch.full((n + off + 4,), 7.0, device=DEV)[off:off + n]
    gpu.dropout_forward(out, x, n, p, SEED, 5, 2)
    same(out, drop(h[0]), "dropout_forward")
    gpu.dropout_residual_forward(out, x, y, n, p, SEED, 5, 2)
    same(out, h[0] + drop(h[1]), "dropout_residual_forward")
    t = a.clone()
    gpu.dropout_backward(t, x, n, p, SEED, 5, 2)
    same(t, h[2] + drop(h[0]), "dropout_backward")
    t, u = a.clone(), b.clone()
    gpu.dropout_residual_backward(t, u, x, n, p, SEED, 5, 2)
    same(t, h[2] + h[0], "dropout_residual_backward dx")
    same(u, h[3] + drop(h[0]), "dropout_residual_backward dy")
    t = a.clone()
    gpu.dropout_residual_backward(t, t, x, n, p, SEED, 5, 2)
    same(t, (h[2] + h[0]) + drop(h[0]), "dropout_residual_backward dx == dy")
    t = x.clone()
    gpu.dropout_forward(t, t, n, p, SEED, 5, 2)
    same(t, drop(h[0]), "dropout_forward in place")
    t = y.clone()
    gpu.dropout_residual_forward(t, x, t, n, p, SEED, 5, 2)
    same(t, h[0] + drop(h[1]), "dropout_residual_forward onto y")
    whole = out._base
    assert (whole[:off] == 7.0).all() and (whole[off + n:] == 7.0).all(), "written outside"


def test_masks_of_step_site_and_seed_differ(gpu):
    n, x = 4096, torch.ones(4096, device=DEV)
    seen = []
    for seed, step, site in ((1, 1, 0), (2, 1, 0), (1, 2, 0), (1, 1, 1), (1 << 40, 1, 0), (1, -1, 2147483647)):
        out = torch.empty(n, device=DEV)
        gpu.dropout_forward(out, x, n, 0.5, seed, step, site)
        same(out, drop_ref.drop(np.ones(n, np.float32), drop_ref.keep(n, 0.5, seed, step, site), 0.5), f"{seed} {step} {site}")
        seen.append(out)
    for i in range(len(seen)):
        for j in range(i):
            assert 0.4 < float((seen[i] != seen[j]).float().mean()) < 0.6


def test_dropped_places_hold_no_trace(gpu):
    """Infinities and NaN in dropped places give +0, in kept places themselves."""
    n = 1000
    kept = torch.from_numpy(drop_ref.keep(n, 0.3, 9, 9, 9)).to(DEV)
    for value in (math.nan, math.inf, -math.inf, -0.0):
        x = torch.full((n,), value, device=DEV)
        out = torch.empty(n, device=DEV)
        gpu.dropout_forward(out, x, n, 0.3, 9, 9, 9)
        assert torch.equal(out[~kept].view(torch.int32), torch.zeros(int((~kept).sum()), dtype=torch.int32, device=DEV))
        assert out[kept].isnan().all() if value != value else (out[kept] == value).all()
        one = torch.ones(n, device=DEV)
        gpu.dropout_residual_forward(out, one, x, n, 0.3, 9, 9, 9)
        assert (out[~kept] == 1.0).all()


SHAPES = [(4, 64, 384), (2, 100, 768), (8, 256, 768), (3, 11, 5), (5, 7, 1030), (2, 33, 1602), (1, 40, 2047), (3, 10, 2048),
          (2, 9, 4097), (1, 7, 8192), (1, 3, 9001), (2, 5, 2), (16, 512, 256), (1, 1, 1), (40, 128, 64)]


@pytest.mark.parametrize("B,T,C", SHAPES)
def test_layernorm_pairs_equal_their_ops(gpu, B, T, C):
    rows, n, p = B * T, B * T * C, 0.25
    x, y, dout = (rand(n, k) for k in range(3))
    w, b = rand(C, 4) * 0.1 + 1.0, rand(C, 5) * 0.1
    e = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    want = [e(n), e(n), e(rows), e(rows)]
    gpu.dropout_residual_forward(want[0], x, y, n, p, SEED, 1, 4)
    gpu.layernorm_forward(want[1], want[2], want[3], want[0], w, b, B, T, C)
    same(want[0], x.cpu().numpy() + drop_ref.drop(y.cpu().numpy(), drop_ref.keep(n, p, SEED, 1, 4), p), "res")
    got = [e(n), e(n), e(rows), e(rows)]
    gpu.dropout_residual_layernorm_forward(*got, x, y, w, b, B, T, C, p, SEED, 1, 4)
    for name, u, v in zip(("res", "out", "mean", "rstd"), got, want):
        assert torch.equal(u, v), name
    start = [rand(n, 6), rand(C, 7), rand(C, 8), rand(n, 9), rand(n, 10)]
    for exact in (False, True):
        gpu.set_layernorm_exact(exact)
        try:
            want_g, got_g = [t.clone() for t in start], [t.clone() for t in start]
            gpu.layernorm_backward(*want_g[:3], dout, want[0], w, want[2], want[3], B, T, C)
            gpu.dropout_residual_backward(want_g[3], want_g[4], want_g[0], n, p, SEED, 1, 4)
            gpu.layernorm_dropout_residual_backward(*got_g, dout, want[0], w, want[2], want[3], B, T, C, p, SEED, 1, 4)
            for name, u, v in zip(("dinp", "dweight", "dbias", "dx", "dy"), got_g, want_g):
                assert torch.equal(u, v), f"{name} exact={exact}"
            one, two = start[3].clone(), start[3].clone()  # dx == dy
            a, b2 = [t.clone() for t in start[:3]], [t.clone() for t in start[:3]]
            gpu.layernorm_backward(*a, dout, want[0], w, want[2], want[3], B, T, C)
            gpu.dropout_residual_backward(one, one, a[0], n, p, SEED, 1, 4)
            gpu.layernorm_dropout_residual_backward(*b2, two, two, dout, want[0], w, want[2], want[3], B, T, C, p, SEED, 1, 4)
            assert torch.equal(one, two), f"dx == dy exact={exact}"
            g2 = [e(n), e(n), e(rows), e(rows)]
            gpu.dropout_residual_layernorm_forward(*g2, x, y, w, b, B, T, C, p, SEED, 1, 4)
            ref = [e(n), e(rows), e(rows)]
            gpu.layernorm_forward(*ref, g2[0], w, b, B, T, C)
            assert torch.equal(g2[0], want[0]) and all(torch.equal(u, v) for u, v in zip(g2[1:], ref))
        finally:
            gpu.set_layernorm_exact(False)


@pytest.mark.parametrize("C", [384, 770])
def test_misaligned_layernorm_pair(gpu, C):
    B, T, p = 3, 21, 0.4
    n, rows = B * T * C, B * T
    for off in (1, 2, 3):
        x, y, w, b = rand(n, 1, off), rand(n, 2, off), rand(C, 3, off), rand(C, 4, off)
        e = lambda k: torch.empty(k + off, device=DEV)[off:]  # noqa: E731
        want, got = [e(n), e(n), e(rows), e(rows)], [e(n), e(n), e(rows), e(rows)]
        gpu.dropout_residual_forward(want[0], x, y, n, p, SEED, 1, 0)
        gpu.layernorm_forward(want[1], want[2], want[3], want[0], w, b, B, T, C)
        gpu.dropout_residual_layernorm_forward(*got, x, y, w, b, B, T, C, p, SEED, 1, 0)
        for u, v in zip(got, want):
            assert torch.equal(u, v)


def test_gradient_against_differences(gpu):
    """The pair's gradient along a direction against central differences of its forward in 64 bits with the same mask:
    off by h^2 of the third derivative (1e-6 of the terms' sizes at h = 1e-4) and (C + rows + 32) 2^-24 of them."""
    B, T, C, p = 2, 6, 96, 0.3
    n, rows = B * T * C, B * T
    x, y, dout, w, b = rand(n, 1), rand(n, 2), rand(n, 3), rand(C, 4), rand(C, 5)
    f = torch.from_numpy(drop_ref.keep(n, p, SEED, 1, 0)).to(DEV).double() / (1 - float(np.float32(p)))

    def forward(x, y):
        r = (x + y * f).view(rows, C)
        var, mean = torch.var_mean(r, 1, correction=0, keepdim=True)
        return (((r - mean) / (var + 1e-5).sqrt() * w.double() + b.double()).view(-1) * dout.double()).sum()

    res, out, mean, rstd = (torch.empty(k, device=DEV) for k in (n, n, rows, rows))
    gpu.dropout_residual_layernorm_forward(res, out, mean, rstd, x, y, w, b, B, T, C, p, SEED, 1, 0)
    dinp, dw, db, dx, dy = (torch.zeros(k, device=DEV) for k in (n, C, C, n, n))
    gpu.layernorm_dropout_residual_backward(dinp, dw, db, dx, dy, dout, res, w, mean, rstd, B, T, C, p, SEED, 1, 0)
    h = 1e-4
    for grad, at in ((dx, 0), (dy, 1)):
        d = rand(n, 20 + at).double()
        v = [x.double(), y.double()]
        fs = []
        for sign in (1, -1):
            t = list(v)
            t[at] = v[at] + sign * h * d
            fs.append(float(forward(*t)))
        size = float((grad.double().abs() * d.abs()).sum())
        assert abs(float((grad.double() * d).sum()) - (fs[0] - fs[1]) / (2 * h)) <= size * (1e-6 + (C + rows + 32) * 2.0 ** -24)


def test_captured_and_replayed(gpu):
    """A captured forward and backward replayed between eager calls of another mask."""
    B, T, C, p = 4, 64, 384, 0.1
    n, rows = B * T * C, B * T
    x, y, dout, w, b = rand(n, 1), rand(n, 2), rand(n, 3), rand(C, 4), rand(C, 5)
    bufs = [torch.empty(k, device=DEV) for k in (n, n, rows, rows)]
    g = [torch.zeros(k, device=DEV) for k in (n, C, C, n, n)]

    def step(fwd, grads, site):
        gpu.dropout_residual_layernorm_forward(*fwd, x, y, w, b, B, T, C, p, SEED, 1, site)
        for t in grads:
            t.zero_()
        gpu.layernorm_dropout_residual_backward(*grads, dout, fwd[0], w, fwd[2], fwd[3], B, T, C, p, SEED, 1, site)

    step(bufs, g, 0)
    want = [t.clone() for t in (*bufs, *g)]
    eager = [torch.empty_like(t) for t in bufs], [torch.empty_like(t) for t in g]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(bufs, g, 0)
        for k in range(3):
            for t in (*bufs, *g):
                t.fill_(2.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, w_) for a, w_ in zip((*bufs, *g), want))
            with torch.cuda.stream(stream):
                step(*eager, 1 + k)
            stream.synchronize()
            assert not torch.equal(eager[0][0], bufs[0])
    finally:
        gpu.set_stream(None)
