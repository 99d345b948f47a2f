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


VOCAB = 50


class PagesOfTokens:
    """A model whose keys are the token ids themselves, kept in the cache's slots: a row's logits depend on what its
    page table finds there, so another request's tokens, or a shifted position, show."""

    def __init__(self):
        self.slots = {}

    def step(self, cache, requests, parts):
        import torch
        cache.grow(requests, [len(p) for p in parts])
        rows = []
        for r, p in zip(requests, parts):
            pages, size = cache.pages[r], cache.page_size
            at = lambda j: (pages[j // size], j % size)  # noqa: E731
            first = cache.lengths[r] - len(p)
            for j, t in enumerate(p):
                self.slots[at(first + j)] = t
                seen = [self.slots[at(u)] for u in range(first + j + 1)]
                rows.append([-((v - 7 * sum(seen) - 3 * len(seen)) % VOCAB) / 9.0 for v in range(VOCAB)])
        return torch.tensor(rows)


@pytest.fixture
def plain_logprobs(monkeypatch):
    import torch
    from trifuse_b200 import ops

    def token_logprobs(logits, tokens, top=0):
        lp = torch.log_softmax(logits.double(), -1)
        best, token = torch.sort(lp, descending=True, stable=True)
        given = torch.where(tokens >= 0, lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], float("nan"))
        return ops.TokenLogprobs(given, None, None, best[:, :top], token[:, :top])

    monkeypatch.setattr(ops, "token_logprobs", token_logprobs)


def batch(n=3):
    from trifuse_b200.paged import Request
    return [Request(list(range(3 + i, 9 + 2 * i)), 2 + i) for i in range(n)]


def answers(requests):
    return [(r.tokens, r.prompt_logprobs, r.logprobs, r.alternatives) for r in requests]


def test_serve_gives_its_pages_back_when_a_step_fails(plain_logprobs):
    """A call that runs out of pages leaves all of them free, and a smaller one on the same cache answers as on a new
    one."""
    from trifuse_b200.paged import serve
    cache, model = small_cache(pages=5), PagesOfTokens()
    with pytest.raises(RuntimeError, match="pages needed"):
        serve(model, cache, batch(3), chunk=4)
    assert state(cache) == (list(range(5)), {}, {})
    got = serve(model, cache, batch(1), chunk=4)
    want = serve(PagesOfTokens(), small_cache(pages=5), batch(1), chunk=4)
    assert answers(got) == answers(want) and state(cache) == (list(range(5)), {}, {})


@pytest.mark.parametrize("others", [[0, 1], [2], [0, 5], ["a"]])
def test_serve_beside_requests_of_the_callers_own(plain_logprobs, others):
    """Requests that the cache holds already keep their tokens, and are not taken for those served."""
    from trifuse_b200.paged import serve
    cache, model = small_cache(pages=30), PagesOfTokens()
    model.step(cache, others, [[40 + i] * 3 for i in range(len(others))])
    kept = {r: list(p) for r, p in cache.pages.items()}
    got = serve(model, cache, batch(3), chunk=4)
    want = serve(PagesOfTokens(), small_cache(pages=30), batch(3), chunk=4)
    assert answers(got) == answers(want)
    assert cache.pages == kept and cache.lengths == {r: 3 for r in others}
    for i, r in enumerate(others):
        assert [model.slots[kept[r][0], j] for j in range(3)] == [40 + i] * 3


@pytest.mark.parametrize("top", [0, 1, 3])
def test_as_many_alternatives_as_asked_for(plain_logprobs, top):
    from trifuse_b200.paged import serve
    for r in serve(PagesOfTokens(), small_cache(pages=30), batch(3), chunk=4, top=top):
        assert [len(a) for a in r.alternatives] == [top] * r.new_tokens == [top] * len(r.tokens)


@pytest.mark.parametrize("chunk", [0, -1, -3])
def test_a_chunk_of_nothing_is_refused(plain_logprobs, chunk):
    from trifuse_b200.paged import serve
    cache, requests = small_cache(), batch(1)
    with pytest.raises(ValueError, match="chunk"):
        serve(PagesOfTokens(), cache, requests, chunk=chunk)
    assert not cache.lengths and answers(requests) == [([], [], [], [])]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_logits_that_are_no_distribution_give_no_token(plain_logprobs, bad):
    """A row with a NaN or +inf, or nothing but -inf, has no next token: told, as the session tells it."""
    from trifuse_b200 import TriFuseError
    from trifuse_b200.paged import serve

    class Bad(PagesOfTokens):
        def step(self, cache, requests, parts):
            logits = super().step(cache, requests, parts)
            if cache.lengths[requests[0]] == 8:
                logits[0, 4 if bad > 0 or bad != bad else slice(None)] = bad
            return logits

    cache, requests = small_cache(), batch(1)  # a prompt of 6
    requests[0].new_tokens = 9
    with pytest.raises(TriFuseError, match="not finite"):
        serve(Bad(), cache, requests, chunk=8)
    assert len(requests[0].tokens) == 2 and not cache.lengths and len(cache.free) == 6


@pytest.mark.parametrize("chunk", [2, 4, 100])
@pytest.mark.parametrize("fails_at", [1, 2, 3, 4])
def test_a_call_that_was_cut_short_may_be_repeated(plain_logprobs, chunk, fails_at):
    """The same requests again: each prompt token's log probability once, and the answers of an undisturbed call."""
    from trifuse_b200.paged import serve

    class Once(PagesOfTokens):
        steps = 0

        def step(self, *a):
            self.steps += 1
            if self.steps == fails_at:
                raise RuntimeError("once")
            return super().step(*a)

    cache, requests, model = small_cache(pages=30), batch(3), Once()
    with pytest.raises(RuntimeError, match="once"):
        serve(model, cache, requests, chunk=chunk)
    got = serve(model, cache, requests, chunk=chunk)
    assert answers(got) == answers(serve(PagesOfTokens(), small_cache(pages=30), batch(3), chunk=chunk))
