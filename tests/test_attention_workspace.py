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
    kept = gpu.scratch_bytes()  # for graphs of other tests
    gpu.reserve(8192, 768)
    assert gpu.scratch_bytes() - kept <= 22 << 20
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


def captured_backward(gpu, n, stream, graphs):
    """A captured attention backward of n single rows of 64 heads: 256 n bytes of workspace. Returns it and its check."""
    x = torch.randn(n, 64, device=DEV)
    lse, g = torch.zeros(n, 64, device=DEV), [torch.zeros(n, 64, device=DEV) for _ in range(3)]
    a = gpu.Attention(nseq=n, NH=64, NKV=64, HS=1, rows_q=n, rows_k=n, max_q=1, max_k=1, scale=0.0)
    call = lambda: gpu.attention_backward_zeroed(*g, x, x, x, x, x, lse, a)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call()  # grows the region
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    graphs.append(graph)

    def check():
        for t in g:
            t.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # one key of weight 1 (a score of 0, and the lse given): dv = dout, to the 2^-23 that two halves hold and a rounding; a
        # scale of 0: dq = dk = 0
        assert ((g[2] - x).abs() <= 2.0 ** -22 * x.abs()).all() and not g[0].any() and not g[1].any()
    check.inputs = (x, lse, g)
    return check


@pytest.mark.gpu
def test_memory_kept_for_graphs_is_counted_bounded_and_released(gpu):
    gpu.set_workspace(None, gpu.Config(B=1, T=1, C=64, V=2, NH=0, maxT=1, L=0))
    gpu.release_graph_memory()
    assert gpu.scratch_bytes() == 0
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    graphs, checks = [], []
    try:
        for i in range(9):
            n = int(2000 * 1.3 ** i)
            checks.append(captured_backward(gpu, n, stream, graphs))
            # the region in use is at most twice what the largest call needs, what is kept for graphs below that again
            assert 256 * n <= gpu.scratch_bytes() <= 4 * (256 * n + 4096)
        held = gpu.scratch_bytes()
        for c in checks + checks[::-1]:
            c()
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            assert gpu.lib.ugk_release_graph_memory() == 1
            torch.zeros(1, device=DEV).add_(1)
        assert gpu.scratch_bytes() == held
        del checks
        graphs.clear()
        gpu.release_graph_memory()
        assert 256 * n <= gpu.scratch_bytes() <= 2 * (256 * n + 4096)
        more = captured_backward(gpu, 4 * n, stream, graphs)  # the region in use was no graph's any more: freed
        assert gpu.scratch_bytes() <= 256 * 4 * n + 4096
        more()
    finally:
        gpu.set_stream(None)
        graphs.clear()
        gpu.release_graph_memory()


def test_release_needs_no_gpu_to_be_declared():
    import ugk
    assert "release_graph_memory" in ugk.__all__ and callable(ugk.release_graph_memory)
