"""The page table of piton_b200.cached_block; no GPU needed."""

import pytest

from piton_b200.cached_block import PageTable


def state(t):
    return list(t.free), list(t.owned), t.host.tolist(), t.table.tolist()


@pytest.mark.parametrize("lengths", [[17, 49], [65, 16], [33, 33]])
def test_a_reservation_that_fails_changes_nothing(lengths):
    t = PageTable(2, 5, 16, 3, "cpu")
    t.reserve([16, 32])
    t.reserve([17])                             # the first sequence alone
    before = state(t)
    with pytest.raises(MemoryError):
        t.reserve(lengths)
    assert state(t) == before
    t.reserve([20, 20])
    assert state(t) == before
    t.reserve([32, 48])
    assert t.owned == [2, 3] and not t.free and t.table.tolist() == t.host.tolist()


def test_released_pages_are_given_out_again():
    t = PageTable(3, 4, 16, 4, "cpu")
    t.reserve([30, 16, 1])
    kept = t.host[1].tolist(), t.host[2].tolist()
    t.release(0)
    assert t.host[0].tolist() == [-1] * 4 and t.table.tolist() == t.host.tolist() and t.owned == [0, 1, 1]
    t.release(0)                                # nothing left to give back
    assert len(t.free) == 2
    t.reserve([0, 16, 48])
    assert t.host[1].tolist() == kept[0] and t.host[2].tolist()[0] == kept[1][0]
    pages = [p for row in t.host.tolist() for p in row if p >= 0]
    assert sorted(pages) == [0, 1, 2, 3] and not t.free
    with pytest.raises(MemoryError):
        t.reserve([1, 16, 48])
    t.release(2)
    t.reserve([33, 16, 0])
    assert t.owned == [3, 1, 0]
