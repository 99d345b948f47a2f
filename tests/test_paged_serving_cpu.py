"""The paged cache's book-keeping and the serving loop around a model of a few lines: what a refused step, a failed
one or a repeated call leaves behind."""
import pytest

from trifuse_b200.paged import PagedCache


def small_cache(pages=6, page=4):
    return PagedCache(1, pages, 1, page, 64, device="cpu")


def state(cache):
    return sorted(cache.free), {r: list(p) for r, p in cache.pages.items()}, dict(cache.lengths)


@pytest.mark.parametrize("requests,counts", [([0, 0], [3, 3]), ([1, 0, 1], [1, 1, 1]), ([0, 1], [2]), ([0], [-1])])
def test_grow_refuses_what_it_cannot_lay_out(requests, counts):
    """A request listed twice would get one part's slots for both, and too few pages."""
    cache = small_cache()
    cache.grow([0], [3])
    before = state(cache)
    with pytest.raises(ValueError):
        cache.grow(requests, counts)
    assert state(cache) == before
