"""Attention's share of the workspace: none where the config has no heads, enough for every shape up to one that has."""
import pytest
import torch

DEV = "cuda"


def test_a_config_without_heads_needs_none():
    """NH 0 is the size without attention; with heads the parts of dk and dv are bounded by their own size."""
    import ugk
    cfg = dict(B=8, T=1024, C=768, V=50257, maxT=1024, L=12)
    without = ugk.workspace_bytes(ugk.Config(NH=0, **cfg))
    # 25 LayerNorm slots of 512 partial rows of 2 C floats, the encoder's 18.7 MB, and what is small beside them
    assert 25 * 512 * 2 * 768 * 4 <= without < 98 << 20
    heads = ugk.workspace_bytes(ugk.Config(NH=12, **cfg)) - without
    # lse and out of the recomputed forward, row sums, 2^17 rows of a head in parts of dk and of dv
    assert heads <= 8192 * 768 * 4 + 2 * 8192 * 12 * 4 + 2 * (1 << 17) * 64 * 4 + 4096
    # heads that the callbacks refuse: 768 floats, 5 that do not divide the channels
    for NH in (1, 5):
        assert ugk.workspace_bytes(ugk.Config(NH=NH, **cfg)) == without
    # small shapes have no parts of dk and dv: 2^15 rows of a head in the forward's parts, and the recomputed forward
    small = dict(B=4, T=64, C=384, V=27, maxT=64, L=6)
    more = ugk.workspace_bytes(ugk.Config(NH=6, **small)) - ugk.workspace_bytes(ugk.Config(NH=0, **small))
    assert more <= (1 << 15) * 66 * 4 + 256 * 384 * 4 + 256 * 6 * 8 + 4096


@pytest.mark.gpu
def test_reserve_without_heads_holds_none(gpu):
    gpu.set_workspace(None, gpu.Config(B=1, T=1, C=64, V=2, NH=0, maxT=1, L=0))
    gpu.reserve(8192, 768)
    assert gpu.scratch_bytes() <= 22 << 20
    x = torch.randn(2 * 64, 3 * 128, device=DEV)
    g, out = torch.zeros_like(x), torch.empty(2 * 64, 128, device=DEV)
    gpu.dense_attention_forward(out, x, 2, 64, 128, 2)
    gpu.dense_attention_backward(g, out, x, 2, 64, 128, 2)  # allocates
    gpu.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("NH,C", [(12, 768), (6, 384), (8, 1024), (5, 40)])
def test_every_shape_up_to_the_config_fits(gpu, NH, C):
    """In a workspace of exactly the config's size: fewer rows (more parts), fewer sequences, grouped heads, one long
    sequence of all rows."""
    B, T, HS = 4, 1024, C // NH
    cfg = gpu.Config(B=B, T=T, C=C, V=50, NH=NH, maxT=T, L=1)
    n = gpu.workspace_bytes(cfg)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=DEV)
    at = (-ws.data_ptr()) % 256
    x = torch.randn(B * T * 3 * C, device=DEV)
    g, out, lse = torch.zeros_like(x), torch.zeros(B * T * C, device=DEV), torch.zeros(B * T * NH, device=DEV)
    try:
        gpu.set_workspace(ws[at:at + n], cfg)
        for b, t in ((B, T), (1, T), (2, T), (1, 300), (4, 128), (1, 1), (4, 700), (3, 511)):
            gpu.dense_attention_forward(out, x, b, t, C, NH)
            gpu.dense_attention_backward(g, out, x, b, t, C, NH)
        for b, t in ((1, B * T), (B, T), (1, 2048), (7, 200), (64, 64), (300, 13)):
            for NKV in {NH, 1, NH // 2 if NH % 2 == 0 else 1}:
                ld = (NH + 2 * NKV) * HS
                a = gpu.Attention(nseq=b, NH=NH, NKV=NKV, HS=HS, rows_q=b * t, rows_k=b * t, max_q=t, max_k=t, ldq=ld, ldk=ld, ldv=ld)
                q, k, v = x, x[NH * HS:], x[(NH + NKV) * HS:]
                gpu.attention_forward(out, lse, q, k, v, a)
                gpu.attention_backward(g, g[NH * HS:], g[(NH + NKV) * HS:], out, q, k, v, out, lse, a)
        gpu.synchronize()
        none = gpu.Config(B=B, T=T, C=C, V=50, NH=0, maxT=T, L=1)
        m = gpu.workspace_bytes(none)
        assert m < n
        gpu.set_workspace(ws[at:at + m], none)
        with pytest.raises(gpu.UgkError, match="attention"):
            gpu.dense_attention_backward(g, out, x, 1, T, C, NH)
    finally:
        gpu.set_workspace(None, cfg)
