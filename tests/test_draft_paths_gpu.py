"""GPU: the ways through the verification that its sizes choose: sums of segments in a launch of their own, also captured and replayed;
many sequences, which sum in theirs; more segments than lanes and segments of several steps; p drawn from where q takes all."""
import pytest
import torch

import cache8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(B, K, V, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    p = torch.rand(B, K + 1, V, generator=g, device=DEV)
    p /= p.sum(2, keepdim=True)
    q = (p[:, :K] * (0.5 + torch.rand(B, K, V, generator=g, device=DEV))).contiguous()
    draft = torch.randint(0, V, (B, K), generator=g, device=DEV).int()
    return p, q, draft, torch.rand(B, K + 1, generator=g, device=DEV)


def call(gpu, p, q, draft, u, out=None):
    B, K1, V = p.shape
    accepted, tokens = out or (torch.full(s, -9, dtype=torch.int32, device=DEV) for s in ((B,), (B, K1)))
    gpu.draft_verify(accepted, tokens, p, q, draft, None, u, B, K1 - 1, V)
    return accepted, tokens


def check(gpu, p, q, draft, u, sample):
    accepted, tokens = call(gpu, p, q, draft, u)
    gpu.synchronize()
    for b in sample:
        a, t = ref.verify(p[b].double().tolist(), None if q is None else q[b].double().tolist(), draft[b].tolist(), draft.shape[1],
                          u[b].double().tolist())
        assert (int(accepted[b]), tokens[b].tolist()) == (a, t), b
    return accepted


@pytest.mark.parametrize("B,V", [(2, 8193), (255, 8193), (256, 8193), (256, 9001), (300, 8192), (2, 300001), (1, 4194305)])
def test_sizes(gpu, B, V):
    p, q, draft, u = case(B, 1, V, V + B)
    sample = sorted({0, 1, B // 2, B - 1} & set(range(B)))
    for x in (0.0, 0.5, 1.0 - 2.0 ** -24):
        u[:, 1] = x
        check(gpu, p, q, draft, u, sample)
    check(gpu, p, None, draft, u, sample)


@pytest.mark.parametrize("B,V", [(3, 300), (3, 20001), (256, 20001), (256, 8192)])
def test_drafts_that_take_all_leave_the_target(gpu, B, V):
    """max(p - q, 0) is 0 throughout: the token is p's, from sums made again."""
    p, q, draft, u = case(B, 1, V, V)
    q[:] = p[:, :1]
    u[:, 0] = 1.0  # refused
    q[1::2] *= 0.5  # every second sequence has something left
    p[1::2].scatter_(2, draft[1::2, :, None].long().expand(-1, 2, -1), 0.0)
    accepted = check(gpu, p, q, draft, u, sorted({0, 1, 2, B // 2, B - 2, B - 1}))
    assert (accepted == 0).all()


@pytest.mark.parametrize("B,V", [(5, 20001), (256, 9001)])
def test_captured(gpu, B, V):
    p, q, draft, u = case(B, 1, V, 9)
    q[::3] = p[::3, :1]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gpu.set_stream(s.cuda_stream)
        try:
            call(gpu, p, q, draft, u)  # its workspace is there
            out = [torch.empty(x, dtype=torch.int32, device=DEV) for x in ((B,), (B, 2))]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call(gpu, p, q, draft, u, out)
            for _ in range(4):
                u.uniform_()
                u[::2, 0] = 1.0
                out[0].fill_(-9)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                eager = call(gpu, p, q, draft, u)
                torch.cuda.synchronize()
                assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
        finally:
            s.synchronize()
            gpu.set_stream(None)
    gpu.synchronize()
