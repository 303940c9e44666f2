"""What a page pool refuses."""
import pytest

from openasr_b200 import backend as bk


def test_positions_that_are_not_held_cannot_be_skipped():
    """extend starts at most where the sequence's pages end, also when that is inside the next page: the
    positions before it would be read without ever having been written"""
    p = bk.KvPool(8, 8, 6, 2)
    s = p.open()
    for start, end in ((1, 2), (5, 8), (7, 20), (8, 9)):
        with pytest.raises(bk.UnsupportedInputs):
            p.extend(s, start, end)
    p.extend(s, 0, 3)  # a whole page is held from here on
    p.extend(s, 3, 8)
    p.extend(s, 8, 13)
    for start, end in ((17, 18), (23, 24), (24, 25)):
        with pytest.raises(bk.UnsupportedInputs):
            p.extend(s, start, end)
    assert p.pages_free() == 6 and (p.table([s])[0] >= 0).sum() == 2
    p.truncate(s, 8)
    with pytest.raises(bk.UnsupportedInputs):
        p.extend(s, 9, 12)
    assert p.extend(s, 8, 12).shape == (0, 2)
