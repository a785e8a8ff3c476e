"""GPU: attention over the cache in 8 bits with scales near the ends of a float's range, of either sign, whose scores are ordinary."""
import pytest
import torch

from test_cache8_gpu import DEV, check, filled, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale,of_q,of_k", [(3.0e38, -90, -40), (2.0e38, -90, -40), (1e-42, 79, 60), (2.0 ** -149, 80, 66), (2.0 ** -126, 66, 60)])
@pytest.mark.parametrize("lq", [1, 5, 20, 100])
def test_scales_at_the_ends_of_the_range(gpu, lq, scale, of_q, of_k, sign):
    NH, NKV, HS, cap = 2, 2, 64, 300

    def size(k, v):
        k *= 2.0 ** of_k
    c, g = filled(gpu, 1, cap, NKV, HS, [cap], size=size)
    q = rand(g, lq, NH, HS) * 2.0 ** of_q
    scale = float(torch.tensor(sign * scale, dtype=torch.float32))  # as a float holds it
    for weigh in (False, True):
        out, L, _ = check(gpu, c, NH, q, [0], [lq], [cap], lq, scale=scale, weigh=weigh)
        assert out.isfinite().all() and float(L.std() if lq > 1 else 1.0) > 1e-3
