"""CPU: what a launch's grid does not hold is refused on the host, by the rows and blocks that there can be."""
import pytest

from test_cache8 import P, shape


def test_more_workgroups_than_a_grid_has():
    import torch
    import ugk
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: they are only safe where no kernel can start")
    lib = ugk.lib
    one = dict(NH=1, NKV=1, q_start=64, q_end=128, table=256, nblocks=8)
    # 128 rows touch three blocks each
    a = shape(ugk, nseq=4_000_000, max_q=128, rows_q=512_000_000, max_k=192, **one)
    for call in (lib.ugk_cache8_store, lib.ugk_cache8_load):
        assert call(*P[:6], a) == 1 and b"exceeds the grid" in lib.ugk_last_error()
    # a workgroup for the weights of 16 blocks
    for nseq, fits in ((65_000, True), (65_100, False)):
        a = shape(ugk, nseq=nseq, max_q=1, rows_q=nseq, max_k=131072, **one)
        assert (lib.ugk_cache8_attention(*P[:8], a) != 1) == fits
        assert fits or b"of their weights" in lib.ugk_last_error()
    # long tables of many sequences alone are no reason
    for nseq, NKV in ((512, 8), (4096, 8), (100_000, 16)):
        a = shape(ugk, nseq=nseq, NH=NKV, NKV=NKV, max_q=1, rows_q=nseq, max_k=131072, q_start=64, q_end=128, table=256, nblocks=8)
        for call, n in ((lib.ugk_cache8_store, 6), (lib.ugk_cache8_load, 6), (lib.ugk_cache8_attention, 7)):
            assert call(*P[:n], *([None] if n == 7 else []), a) != 1
