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


def model_that(forward, vocab=50):
    from trifuse_b200.model import Config
    from trifuse_b200.paged import PagedOLMoE
    model = object.__new__(PagedOLMoE)
    model.cfg = Config(layers=1, vocab=vocab)
    model._forward = forward
    return model


@pytest.mark.parametrize("error", [ValueError, RuntimeError, KeyboardInterrupt])
def test_a_step_that_raises_leaves_the_cache_as_it_was(error):
    """Token ids past the vocabulary, a launch that fails: no token that was never written is counted."""
    def fail(*a):
        raise error("no")

    cache = small_cache()
    fine, failing = model_that(lambda cache, requests, tokens, counts: list(requests)), model_that(fail)
    for requests, parts in (([7], [[1] * 5]), ([7, 8], [[1], [2] * 3]), ([8, 9, 7], [[1] * 2, [], [3] * 4])):
        before, order = state(cache), list(cache.free)
        with pytest.raises(error):
            failing.step(cache, requests, parts)
        assert state(cache) == before and cache.free == order
        assert fine.step(cache, requests, parts) == requests
    assert cache.lengths == {7: 10, 8: 5, 9: 0}


def test_a_step_that_cannot_run_leaves_the_cache_as_it_was():
    """The model's own forward, which raises here at its first look for a device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("raises only where there is no device")
    from trifuse_b200.model import Config
    from trifuse_b200.paged import PagedOLMoE
    model = object.__new__(PagedOLMoE)
    model.cfg = Config(layers=1, heads=1, kv_heads=1, head_dim=64, vocab=50)
    cache = small_cache()
    with pytest.raises(Exception):
        model.step(cache, [0, 1], [[1] * 5, [2]])
    assert state(cache) == (list(range(6)), {}, {})
