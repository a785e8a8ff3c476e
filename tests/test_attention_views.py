"""What the binding takes as rows: views whose rows are the call's stride apart, and no others."""
import pytest
import torch

import ugk

NH, HS, C = 4, 16, 64
ROWS = 24


class FakeCuda(torch.Tensor):
    """A host tensor that says it is on the GPU, for the checks that come before a call."""
    @property
    def device(self):
        return torch.device("cuda", 0)


def rows(x, ld=C, w=C, need=None, heads=NH):
    x = x.as_subclass(FakeCuda)
    return ugk._rows_ptr_or_raise(x, "q", (ROWS - 1) * ld + w if need is None else need, ld, w, heads)


@pytest.fixture(autouse=True)
def one_device(monkeypatch):
    ugk._import_torch()
    monkeypatch.setattr(ugk, "_one_device", True)


def test_views_that_hold_the_rows():
    buf = torch.zeros(ROWS, 3 * C)
    assert rows(buf[:, C:2 * C], 3 * C) == buf.data_ptr() + 4 * C
    assert rows(buf.view(ROWS, 3, NH, HS)[:, 2], 3 * C) == buf.data_ptr() + 8 * C
    assert rows(buf.view(2, ROWS // 2, 3 * C)[:, :, :C], 3 * C) == buf.data_ptr()
    assert rows(buf.view(-1)[C:], 3 * C) == buf.data_ptr() + 4 * C  # flat, from the first element on
    assert rows(buf, 3 * C) == buf.data_ptr()
    assert rows(buf[:, :HS], 3 * C) == buf.data_ptr()  # the first head of each row
    cache = torch.zeros(3, 8, C)
    for n in (1, 2, 8):  # the filled part of a cache, its offsets those of the whole
        assert rows(cache[:, :n]) == cache.data_ptr()
    split = cache.view(3, 8, NH, HS)
    for n in (1, 5):
        assert rows(split[:, :n]) == cache.data_ptr()
    one = torch.zeros(ROWS, 6, HS)[:, 4:5]  # the one key head of rows that hold four query heads and a value head too
    assert rows(one, 6 * HS, HS, need=0, heads=1) == one.data_ptr()
    assert rows(cache[1:2], need=0) == cache.data_ptr() + 4 * 8 * C
    wide = torch.zeros(ROWS, C + 5)
    assert rows(wide[:, :C], C + 5) == wide.data_ptr()
    assert rows(wide.as_strided((ROWS, NH, HS), (C + 5, HS, 1)), C + 5) == wide.data_ptr()


@pytest.mark.parametrize("name", ["exchanged", "another stride", "expanded heads", "expanded rows", "every other row", "heads apart", "one head"])
def test_views_that_do_not(name):
    buf = torch.zeros(2 * ROWS, 3 * C)
    x, ld = {
        "exchanged": (torch.zeros(ROWS, NH, HS).transpose(0, 1), C),
        "another stride": (buf[:ROWS, :C], C),
        "expanded heads": (torch.zeros(ROWS, 1, HS).expand(ROWS, NH, HS), C),
        "expanded rows": (torch.zeros(1, C).expand(ROWS, C), C),
        "every other row": (buf[::2], 3 * C),
        "heads apart": (torch.zeros(ROWS, NH, 2 * HS)[:, :, :HS], 2 * C),
        "one head": (torch.zeros(ROWS, 6, C)[:, 4:5], C),
    }[name]
    with pytest.raises(ValueError, match="does not hold rows of 64 floats"):
        rows(x, ld, need=0, heads=1 if name == "one head" else NH)


def test_elements_apart():
    with pytest.raises(ValueError, match="last stride"):
        rows(torch.zeros(C, ROWS).t(), need=0)
