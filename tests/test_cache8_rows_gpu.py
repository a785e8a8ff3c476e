"""GPU: rows of the attention over the cache in 8 bits that see no key, whatever their q holds."""
import math

import pytest
import torch

from test_cache8_gpu import DEV, attend, filled, place_rows, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [200, 2600])
@pytest.mark.parametrize("lq,lk", [(3, 1), (8, 3), (20, 6), (40, 9), (100, 70)])
def test_rows_without_a_key_are_zero_whatever_they_hold(gpu, lq, lk, cap):
    """More rows than keys: the first rows see nothing, also those that are no numbers; a row that sees some is NaN by its own alone."""
    NH, NKV, HS = 2, 2, 64
    lens, keys = [lq, 2], [lk, cap]
    c, g = filled(gpu, 2, cap, NKV, HS, keys)
    starts, rows = place_rows(lens)
    q = rand(g, rows, NH, HS)
    for weigh in (False, True):
        w0, w = (torch.zeros(c.table.shape, device=DEV) if weigh else None for _ in "ab")
        want, L0 = attend(gpu, c, NH, q, starts, lens, keys, rows, weight=w0)
        bad, none = q.clone(), lq - lk
        bad[starts[0], 0, 3], bad[starts[0] + none - 1, 1, 5] = math.nan, -math.inf
        bad[starts[0]:starts[0] + none, 0, 7] = math.inf
        out, L = attend(gpu, c, NH, bad, starts, lens, keys, rows, weight=w)
        gpu.synchronize()
        at = slice(starts[0], starts[0] + none)
        assert (out[at] == 0).all() and (L[at] == -math.inf).all()
        assert torch.equal(out, want) and torch.equal(L, L0)
        assert not weigh or torch.equal(w, w0)
