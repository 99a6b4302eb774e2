"""Pages with several holders that come back in one list."""
import pytest

from gpullama3.java_b200.cache.pages import CacheError, PagePool


def test_a_page_given_back_twice_by_two_holders_is_free_once():
    pool = PagePool(6)
    a, b, c = pool.alloc(3)
    pool.share([b])
    pool.free([b, a, b])
    assert pool.n_free == 5 and pool.n_held == 1 and pool.n_shared == 0
    out = pool.alloc(5)
    assert sorted(out + [c]) == list(range(6))


def test_a_page_given_back_twice_that_another_still_holds_is_not_free():
    pool = PagePool(3)
    p, = pool.alloc(1)
    pool.share([p])
    pool.share([p])
    pool.free([p, p])
    assert pool.n_free == 2 and pool.holders(p) == 1 and pool.n_shared == 0
    pool.free([p])
    assert pool.n_free == 3


@pytest.mark.parametrize("pages", [[0, 0, 0], [0, 2], [1, 3], [-1]])
def test_a_list_that_is_refused_changes_nothing(pages):
    pool = PagePool(3)
    assert sorted(pool.alloc(2)) == [0, 1]
    pool.share([0])
    with pytest.raises(CacheError):
        pool.free(pages)
    with pytest.raises(CacheError):
        pool.share([1, 2])
    assert pool.n_free == 1 and pool.n_shared == 1 and [pool.holders(p) for p in range(3)] == [2, 1, 0]
    pool.free([0, 1, 0])
    assert pool.n_free == 3 and pool.n_shared == 0
