"""CPU: what the entry points of the cache in 8 bits and of the drafts refuse on the host, and the plain forms of their tests."""
import ctypes
import math

import pytest
import torch

import cache8_ref as ref

P = [1 << 20 | 256 * i for i in range(9)]


def shape(ugk, **kw):
    base = dict(nseq=2, NH=4, NKV=2, HS=64, rows_q=10, max_q=5, max_k=130, nblocks=6)
    base.update(kw)
    return ugk.Cache8(**base)


def calls(lib, a, p=P):
    yield lambda: lib.ugk_cache8_store(*p[:6], a)
    yield lambda: lib.ugk_cache8_load(*p[:6], a)
    yield lambda: lib.ugk_cache8_attention(*p[:8], a)


REFUSED = [
    (dict(nseq=-1), ">= 0"), (dict(rows_q=-1), ">= 0"), (dict(max_q=-1), ">= 0"), (dict(max_k=-1), ">= 0"), (dict(nblocks=-1), ">= 0"),
    (dict(NH=0), "divide"), (dict(NKV=0), "divide"), (dict(NKV=3), "divide"), (dict(NKV=-2), "divide"),
    (dict(HS=0), "HS must be"), (dict(HS=129), "HS must be"), (dict(scale=math.nan), "finite"), (dict(scale=math.inf), "finite"),
    (dict(q_start=64), "together"), (dict(q_end=64), "together"), (dict(rows_q=11), "nseq"), (dict(nblocks=5), "nblocks"),
    (dict(ld_table=2), "ld_table"), (dict(ld_table=4), "nblocks"), (dict(ldq=255), "stride"), (dict(ldk=127), "stride"),
    (dict(ldv=-1), "stride"), (dict(ldo=1), "stride"), (dict(ldk=1 << 59), "address space"),
    (dict(NH=1 << 26, NKV=1 << 26, HS=128), "INT_MAX"), (dict(max_k=(1 << 30) + 1, table=64), "2^30"),
    (dict(nseq=1, NH=128, max_q=1 << 25, rows_q=1 << 25), "2^30"),
    (dict(nseq=1 << 16, NH=512, NKV=512, HS=4, max_q=1, rows_q=1 << 16, nblocks=1 << 30, max_k=64), "grid"),
]


@pytest.mark.parametrize("change,text", REFUSED)
def test_shapes_refused_on_the_host(change, text):
    import ugk
    for call in calls(ugk.lib, shape(ugk, **change)):
        assert call() == 1 and text.encode() in ugk.lib.ugk_last_error()


def test_pointers_refused_on_the_host():
    import ugk
    lib, a = ugk.lib, shape(ugk)
    for n, call in ((6, lib.ugk_cache8_store), (6, lib.ugk_cache8_load), (8, lib.ugk_cache8_attention)):
        for i in range(n):
            if n == 8 and i in (1, 7):
                continue  # lse and weight may be NULL
            x = list(P[:n])
            x[i] = None
            assert call(*x, a) == 1 and b"NULL" in lib.ugk_last_error()
    for call, odd in ((lib.ugk_cache8_store, 0), (lib.ugk_cache8_store, 2), (lib.ugk_cache8_load, 4), (lib.ugk_cache8_attention, 5)):
        x = list(P[:8 if call is lib.ugk_cache8_attention else 6])
        x[odd] += 8
        assert call(*x, a) == 1 and b"aligned" in lib.ugk_last_error()
    for call, i, j in ((lib.ugk_cache8_store, 0, 2), (lib.ugk_cache8_store, 1, 3), (lib.ugk_cache8_load, 0, 1), (lib.ugk_cache8_attention, 0, 2)):
        x = list(P[:8 if call is lib.ugk_cache8_attention else 6])
        x[i] = x[j]
        assert call(*x, a) == 1 and b"distinct" in lib.ugk_last_error()
    many = shape(ugk, nseq=1, max_q=129, rows_q=129, nblocks=3)
    assert lib.ugk_cache8_attention(*P[:8], many) == 1 and b"256 rows" in lib.ugk_last_error()


def test_weights_of_more_workgroups_than_a_grid_has():
    import ugk
    a = shape(ugk, nseq=2000000, NH=1, NKV=1, rows_q=256, max_q=256, max_k=64, nblocks=8, q_start=64, q_end=128, table=256, ld_table=1)
    x = list(P[:8])
    assert ugk.lib.ugk_cache8_attention(*x, a) == 1 and b"grid" in ugk.lib.ugk_last_error()


def test_the_structure_holds_what_it_was_given():
    import ugk
    given = dict(nseq=3, NH=8, NKV=2, HS=50, rows_q=11, max_q=7, max_k=130, nblocks=9, causal=False, scale=0.5, q_start=64, q_end=128,
                 k_len=192, table=256, ld_table=5, ldq=400, ldk=1 << 40, ldv=101, ldo=402)
    a = ugk.Cache8(**given)
    for name, value in given.items():
        assert getattr(a, name) == value, name
    b = ugk.Cache8(1, 1, 1, 64, 1, 1, 64, 1)
    assert (b.q_start, b.q_end, b.k_len, b.table, b.ld_table, b.ldq, b.causal, b.scale) == (None, None, None, None, 0, 0, 1, 0.125)
    with pytest.raises(TypeError):
        ugk.Cache8(1, 1, 1, 64, 1, 1, 64, 1.5)


def test_nothing_to_do_is_done_without_a_gpu():
    import ugk
    lib = ugk.lib
    for kw in (dict(nseq=0, rows_q=0), dict(max_q=0, rows_q=0)):
        for call in calls(lib, shape(ugk, **kw), [None] * 9):
            assert call() == 0
    assert lib.ugk_cache8_store(*[None] * 6, shape(ugk, max_k=0)) == 0
    assert lib.ugk_cache8_evict(*[None] * 7, 0, 5, 3, 0, 1) == 0 and lib.ugk_cache8_evict(*[None] * 7, 5, 0, 3, 0, 1) == 0
    assert lib.ugk_draft_verify(*[None] * 7, 0, 4, 27) == 0


def test_evict_and_verify_refused_on_the_host():
    import ugk
    lib = ugk.lib
    for sizes, text in (((-1, 8, 4, 1, 1), b">= 0"), ((2, -8, 4, 1, 1), b">= 0"), ((2, 16385, 4, 1, 1), b"at most 16384"),
                        ((1 << 22, 8, 4, 1, 1), b"grid"), ((2, 8, 4, -1, 1), b"first"), ((2, 8, 4, 1, 0), b"recent"),
                        ((2, 8, 4, 3, 2), b"keep"), ((2, 8, 0, 0, 1), b"keep"), ((2, 8, 1, 2 ** 31 - 1, 2), b"keep")):
        assert lib.ugk_cache8_evict(*P[:7], *sizes) == 1 and text in lib.ugk_last_error(), sizes
    for i in range(7):
        x = list(P[:7])
        x[i] = None
        assert lib.ugk_cache8_evict(*x, 2, 8, 4, 1, 1) == 1 and b"NULL" in lib.ugk_last_error()
    for i, j in ((0, 1), (0, 2), (0, 3), (1, 2), (2, 3), (0, 5), (0, 6), (1, 4), (1, 6), (2, 4), (2, 5), (3, 4), (3, 5), (3, 6)):
        x = list(P[:7])
        x[i] = x[j]
        assert lib.ugk_cache8_evict(*x, 2, 8, 4, 1, 1) == 1 and b"own input" in lib.ugk_last_error(), (i, j)
    for sizes, text in (((-1, 4, 27), b">= 0"), ((2, -1, 27), b">= 0"), ((2, 4, 0), b"V > 0"), ((1 << 22, 4, 27), b"grid"),
                        ((1 << 20, 1 << 12, 27), b"grid"), ((2, 4, (1 << 30) + 1), b"2^30")):
        assert lib.ugk_draft_verify(*P[:7], *sizes) == 1 and text in lib.ugk_last_error(), sizes
    for i in (0, 1, 2, 4, 6):
        x = list(P[:7])
        x[i] = None
        assert lib.ugk_draft_verify(*x, 2, 4, 27) == 1 and b"NULL" in lib.ugk_last_error()
    for i, j in ((0, 1), (0, 4), (1, 4), (0, 5), (1, 5)):
        x = list(P[:7])
        x[i] = x[j]
        assert lib.ugk_draft_verify(*x, 2, 4, 27) == 1 and b"distinct" in lib.ugk_last_error()


def test_tensors_refused_by_the_binding():
    import ugk
    with pytest.raises(ValueError, match="on the GPU"):
        shape(ugk, k_len=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="on the GPU"):
        ugk.cache8_store(torch.zeros(1, dtype=torch.int8), 0, 0, 0, 0, 0, shape(ugk))
    with pytest.raises(TypeError):
        ugk.cache8_attention(0, 0, 0, "k8", 0, 0, 0, shape(ugk))
    with pytest.raises(ValueError, match="on the GPU"):
        ugk.draft_verify(torch.zeros(2, dtype=torch.int32), 0, 0, 0, 0, 0, 0, 2, 4, 27)
    with pytest.raises(ValueError, match="on the GPU"):
        ugk.cache8_evict(torch.zeros(16, dtype=torch.int32), 0, 0, 0, 0, 0, 0, 2, 8, 4)
    a = shape(ugk, table=64, ld_table=3)
    assert a.ld_table == 3 and abs(a.scale - 0.125) < 1e-9


def test_bytes_of_a_cache():
    import ugk
    assert ctypes.sizeof(ugk.Cache8) % 8 == 0
    for HS, HP in ((1, 16), (16, 16), (17, 32), (50, 64), (64, 64), (80, 80), (128, 128)):
        assert ugk.cache8_bytes(7, 3, HS) == 7 * 3 * 64 * HP
    assert ugk.cache8_bytes(1 << 20, 64, 128) == 1 << 39
    for bad in ((-1, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 129)):
        assert ugk.cache8_bytes(*bad) == 0


def test_model_holds_what_was_stored_to_a_step():
    """Rows stored whole are off by half a step at most, those of a block whose scale was raised later by less than a whole one."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(150, 2, 8, generator=g) * torch.exp2(torch.randint(-3, 4, (150, 1, 1), generator=g).float())
    whole, pieces = ref.Model(2, 8), ref.Model(2, 8)
    whole.store(x, 150)
    for i in range(150):
        pieces.store(x[i:i + 1], i + 1)
    for m, most in ((whole, 0.5), (pieces, 1.0)):
        s = torch.stack(m.scales).repeat_interleave(64, 0)[:150, :, None]
        assert ((m.values() - x).abs() <= most * s).all()
    assert torch.equal(torch.stack(whole.scales), torch.stack(pieces.scales))
    top = torch.stack([x[j:j + 64].abs().amax((0, 2)) for j in (0, 64, 128)]).double()
    s = torch.stack(whole.scales)
    assert (top <= 127 * s).all() and (top > 63.5 * s).all()


def test_scales_of_the_reference():
    assert ref.scale_for(127.0) == 1.0 and ref.scale_for(127.00001) == 2.0 and ref.scale_for(63.5) == 0.5
    assert ref.scale_for(0.0) == 0.0 and ref.scale_for(1e-44) == 2.0 ** -126 and ref.scale_for(3.4e38) == 2.0 ** 121


def test_verify_of_the_reference_keeps_the_targets_distribution():
    """Summed over the drafts' distribution and a fine grid of random numbers, tokens come as the target has them."""
    p, q = [0.5, 0.125, 0.375], [0.25, 0.5, 0.25]
    grid = [(i + 0.5) / 64 for i in range(64)]
    got = [0.0] * 3
    for t in range(3):
        for u0 in grid:
            for u1 in grid:
                a, tokens = ref.verify([p, p], [q], [t], 1, [u0, u1])
                got[tokens[0]] += q[t] / 64 ** 2
    assert all(abs(x - y) < 0.01 for x, y in zip(got, p))


def test_attention_of_the_reference_at_a_known_point():
    q, k, v = torch.zeros(2, 1, 4), torch.zeros(3, 1, 4), torch.arange(12.0).view(3, 1, 4)
    out, lse, weight, tol, *_ = ref.attention(q, k, v, 1.0, True, True)
    assert torch.allclose(out[:, 0], torch.stack((v[:2].mean(0)[0], v.mean(0)[0])).double())
    assert torch.allclose(lse[:, 0], torch.log(torch.tensor([2.0, 3.0], dtype=torch.float64))) and abs(float(weight) - 2) < 1e-12
    assert (tol < 1e-4).all()
