"""CPU: what the attention entry points refuse on the host, and the 64-bit reference of their tests."""
import ctypes
import math

import pytest
import torch

import att_ref
from att_ref import Seqs


def shape(ugk, **kw):
    base = dict(nseq=2, NH=4, NKV=2, HS=64, rows_q=10, rows_k=10, max_q=5, max_k=5)
    base.update(kw)
    return ugk.Attention(**base)


REFUSED = [
    (dict(nseq=-1), "must be >= 0"), (dict(rows_q=-1), "must be >= 0"), (dict(max_k=-4), "must be >= 0"),
    (dict(NH=0), "divide"), (dict(NKV=0), "divide"), (dict(NKV=3), "divide"), (dict(NKV=-2), "divide"),
    (dict(HS=0), "HS must be"), (dict(HS=129), "HS must be"), (dict(scale=math.nan), "finite"), (dict(scale=math.inf), "finite"),
    (dict(q_start=64), "together"), (dict(k_end=64), "together"), (dict(rows_q=11), "nseq"), (dict(rows_k=9), "nseq"),
    (dict(ldq=255), "stride"), (dict(ldk=127), "stride"), (dict(ldv=-1), "stride"), (dict(ldo=1), "stride"),
    (dict(ldk=1 << 59), "address space"), (dict(nseq=1, NH=128, max_q=1 << 25, rows_q=1 << 25, max_k=10), "2^30"),
    (dict(nseq=1 << 20, NH=2048, max_q=1, rows_q=1 << 20, max_k=1 << 10, rows_k=1 << 30, HS=4, NKV=2048), "grid"),
    (dict(NH=1 << 26, NKV=1 << 26, HS=128), "INT_MAX"),
]


@pytest.mark.parametrize("change,text", REFUSED)
def test_shapes_refused_on_the_host(change, text):
    import ugk
    a = shape(ugk, **change)
    lib, p = ugk.lib, [1 << 20 | 256 * i for i in range(9)]
    assert lib.ugk_attention_forward(*p[:5], a) == 1
    assert text.encode() in lib.ugk_last_error()
    assert lib.ugk_attention_backward(*p, a) == 1 and text.encode() in lib.ugk_last_error()
    assert lib.ugk_attention_backward_zeroed(*p, a) == 1 and text.encode() in lib.ugk_last_error()


def test_pointers_refused_on_the_host():
    import ugk
    lib, a = ugk.lib, shape(ugk)
    p = [1 << 20 | 256 * i for i in range(9)]
    for i in (0, 2, 3, 4):
        x = list(p[:5])
        x[i] = None
        assert lib.ugk_attention_forward(*x, a) == 1 and b"NULL" in lib.ugk_last_error()
    for i in range(9):
        x = list(p)
        x[i] = None
        assert lib.ugk_attention_backward(*x, a) == 1 and b"NULL" in lib.ugk_last_error()
    for i in (2, 3, 4):
        x = list(p[:5])
        x[0] = x[i]
        assert lib.ugk_attention_forward(*x, a) == 1 and b"distinct" in lib.ugk_last_error()
    for i, j in ((0, 1), (1, 2), (0, 3), (1, 5), (2, 6), (0, 7), (2, 8)):
        x = list(p)
        x[i] = x[j]
        assert lib.ugk_attention_backward(*x, a) == 1 and b"distinct" in lib.ugk_last_error()
    # nothing to compute succeeds without a GPU
    assert lib.ugk_attention_forward(None, None, None, None, None, shape(ugk, nseq=0, rows_q=0, rows_k=0)) == 0
    assert lib.ugk_attention_forward(None, None, None, None, None, shape(ugk, rows_q=0, max_q=0)) == 0
    assert lib.ugk_attention_backward(*[None] * 9, shape(ugk, nseq=0, rows_q=0, rows_k=0)) == 0
    assert lib.ugk_dense_attention_forward(None, 256, 512, 2, 3, 64, 5) == 1 and b"multiple" in lib.ugk_last_error()
    assert lib.ugk_dense_attention_forward(None, 256, 512, -2, 3, 64, 4) == 1
    assert lib.ugk_dense_attention_forward(None, 256, 512, 2, 3, 516, 4) == 1 and b"HS" in lib.ugk_last_error()
    assert lib.ugk_dense_attention_backward(None, 256, 512, 256, 2, 3, 64, 4) == 1 and b"distinct" in lib.ugk_last_error()
    assert lib.ugk_dense_attention_backward(None, None, None, None, 0, 3, 64, 4) == 0
    assert lib.ugk_last_error() == b""


def test_binding_refuses_tensors_it_cannot_use():
    import ugk
    a = shape(ugk)
    t = torch.zeros(10, 256)
    with pytest.raises(ValueError, match="on the GPU"):
        ugk.attention_forward(t, None, t, t, t, a)
    with pytest.raises(TypeError, match="expected a torch tensor"):
        ugk.attention_forward(t, None, [1.0], t, t, a)
    with pytest.raises(ValueError, match="on the GPU"):
        shape(ugk, q_start=torch.zeros(2, dtype=torch.int32))


def test_struct_matches_the_header():
    import ugk
    assert ctypes.sizeof(ugk.Attention) == 9 * 4 + 4 + 4 * 8 + 4 * 8
    assert ugk.Attention.scale.offset == 36 and ugk.Attention.ldo.offset == 96
    assert shape(ugk).scale == pytest.approx(0.125)


def test_reference_against_autograd():
    """The reference's gradient against torch's in 64 bits, its forward against a plain softmax, its empty rows."""
    g = torch.Generator().manual_seed(1)
    s = Seqs([5, 0, 9], [7, 3, 4], gap=1, tail=2)
    q = torch.randn(s.rows_q, 4, 8, generator=g, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(s.rows_k, 2, 8, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    dout = torch.randn(s.rows_q, 4, 8, generator=g, dtype=torch.float64)
    out, lse, tol, tol_l = att_ref.forward(s, q, k, v, 0.3, True)
    total = 0.0
    for b in range(3):
        for h in range(4):
            x, y, z = q[s.q[b]:s.q[b] + s.lq[b], h], k[s.k[b]:s.k[b] + s.lk[b], h // 2], v[s.k[b]:s.k[b] + s.lk[b], h // 2]
            ok = att_ref.allowed(s.lq[b], s.lk[b], True)
            full = ok.any(1)
            P = torch.softmax((x @ y.T * 0.3).masked_fill(~ok, -math.inf)[full], 1)
            o = P @ z
            rows = torch.arange(s.q[b], s.q[b] + s.lq[b])[full]
            assert torch.allclose(out[rows, h], o, rtol=1e-12, atol=1e-12)
            total = total + (o * dout[rows, h]).sum()
    assert (out[s.q[2]:s.q[2] + 5] == 0).all() and (lse[s.q[2]:s.q[2] + 5] == -math.inf).all()
    total.backward()
    got, _ = att_ref.backward(s, q.detach(), k.detach(), v.detach(), out.detach(), lse.detach(), dout, 0.3, True)
    for x, t in zip(got, (q, k, v)):
        assert torch.allclose(x, t.grad, rtol=1e-9, atol=1e-9)
    assert (tol[~out.isnan()] < 1e-4).all() and tol_l[~lse.isnan()].isfinite().all()


def test_more_sequences_than_the_offsets_hold():
    import ugk
    a = shape(ugk)
    a.nseq = 1 << 20  # no offset tensors: the library's own checks apply
    t = torch.zeros(10, 256)
    with pytest.raises(ValueError, match="on the GPU"):
        ugk.attention_forward(t, None, t, t, t, a)
    a._most = 2
    with pytest.raises(ValueError, match="the offsets hold 2"):
        ugk.attention_forward(t, None, t, t, t, a)
    with pytest.raises(ValueError, match="the offsets hold 2"):
        ugk.attention_backward(t, t, t, t, t, t, t, t, t, a)
