"""Eviction with few free pages, on a device made of host memory: it takes the new pages before it gives back the old, so sequences that
find no room together are cut one call each, and a pool without free pages cuts nothing."""
from tests.test_paged_evict import Weighted, ints, shim  # noqa: F401

NOMEM = -7


def test_one_sequence_a_call_where_few_pages_are_free(shim):  # noqa: F811
    s = Weighted(shim)
    assert s.begin([0], [97]) == 0
    s.write()
    assert s.begin([1, 2], [70, 30]) == 0
    s.write()
    assert s.begin([2], [66]) == 0  # 4, 3 and 3 pages of 12: 2 are free
    s.write()
    before = s.state()
    assert before[2] == 2 and s.evict([0, 1, 2], [41, 50, 64], 1, 40) == NOMEM and s.state() == before
    s.whole()
    for x, keep in ((0, 41), (1, 50), (2, 64)):
        assert s.evict([x], [keep], 1, 40) == 0
        s.cut(x, keep, 1, 40)
        s.whole()
    assert s.state()[2] == 6
    s.close()


def test_a_full_pool_cuts_nothing(shim):  # noqa: F811
    s = Weighted(shim)
    assert s.begin([0], [100]) == 0 and shim.mpg_reserve(s.h, 2, ints([1, 2]), ints([250, 0])) == 0
    s.write()
    before = s.state()
    assert before[2] == 0 and s.evict([0], [41], 0, 40) == NOMEM and s.state() == before
    s.whole()
    assert shim.mpg_free(s.h, 1, ints([1])) == 0
    s.content[1], s.weights[1] = [], []
    assert s.evict([0], [41], 0, 40) == 0
    s.cut(0, 41, 0, 40)
    s.whole()
    s.close()
