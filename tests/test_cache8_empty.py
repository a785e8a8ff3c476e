"""CPU: a cache without blocks is refused where its blocks would be read."""
import pytest

from test_cache8 import P, shape


def test_attention_over_no_blocks_is_refused():
    """Numbers of blocks that are not there are masked, and block 0 is read in their place: there has to be one."""
    import torch
    import ugk
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: they are only safe where no kernel can start")
    lib = ugk.lib
    for kw in (dict(), dict(max_k=1), dict(NH=2, max_q=100, rows_q=200)):
        a = shape(ugk, nblocks=0, table=256, **kw)
        for weight in (None, P[7]):
            assert lib.ugk_cache8_attention(*P[:7], weight, a) == 1 and b"nblocks" in lib.ugk_last_error()
    # nothing to read: rows of no keys, no rows
    assert lib.ugk_cache8_attention(*P[:8], shape(ugk, nblocks=0, max_q=0, rows_q=0, table=256)) == 0
    assert lib.ugk_cache8_attention(*P[:8], shape(ugk, nblocks=0, max_k=0, table=256)) != 1
