"""CPU: outputs of the verification that are also its inputs are refused."""
import pytest

from test_cache8 import P


@pytest.mark.parametrize("out", [0, 1])
@pytest.mark.parametrize("inp", [2, 3, 4, 5, 6])
def test_an_output_that_is_an_input_is_refused(out, inp):
    import torch
    import ugk
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: they are only safe where no kernel can start")
    x = list(P[:7])
    x[inp] = x[out]
    assert ugk.lib.ugk_draft_verify(*x, 2, 4, 27) == 1 and b"distinct" in ugk.lib.ugk_last_error()
    x = list(P[:7])
    x[3] = x[5] = None  # may be NULL, both at once
    assert ugk.lib.ugk_draft_verify(*x, 2, 4, 27) != 1
