"""The paged cache's page lists when requests share pages: what every request reads back after any sequence of steps,
and which pages are free."""
import random

import pytest
import torch

from trifuse_b200 import ops
from trifuse_b200.paged import Hypothesis, PagedCache, beam_search


@pytest.fixture
def copies(monkeypatch):
    """paged_copy on the CPU; the pairs of each call."""
    calls = []

    def copy(arrays, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for t in arrays:
            t[:, dst] = t[:, src]
        calls.append(list(zip(src, dst)))

    monkeypatch.setattr(ops, "paged_copy", copy)
    return calls


class Book:
    """A cache whose requests' tokens are numbers, written where the cache says and read back."""

    def __init__(self, pages=40, page=4, layers=2):
        self.cache = PagedCache(layers, pages, 1, page, 64, device="cpu")
        self.said = {}
        self.next = 1

    def grow(self, requests, counts):
        c = self.cache
        before = {r: c.lengths.get(r, 0) for r in requests}
        c.grow(requests, counts)
        for r, n in zip(requests, counts):
            self.said.setdefault(r, [])
            for t in range(before[r], before[r] + n):
                for l in range(c.k.shape[0]):
                    c.k[l, c.pages[r][t // c.page_size], 0, t % c.page_size, 0] = self.next % 2000
                    c.v[l, c.pages[r][t // c.page_size], 0, t % c.page_size, 0] = l
                self.said[r].append(self.next % 2000)
                self.next += 1

    def check(self):
        c = self.cache
        assert c.lengths == {r: len(t) for r, t in self.said.items()}
        for r, tokens in self.said.items():
            assert len(c.pages[r]) == -(-len(tokens) // c.page_size)
            for l in range(c.k.shape[0]):
                got = [float(c.k[l, c.pages[r][t // c.page_size], 0, t % c.page_size, 0]) for t in range(len(tokens))]
                assert got == tokens
        listed = [p for pages in c.pages.values() for p in pages]
        assert sorted(c.free + list(set(listed))) == list(range(c.k.shape[1])) and not set(c.free) & set(listed)
        assert c.shares == {p: listed.count(p) for p in set(listed) if listed.count(p) > 1}


@pytest.mark.parametrize("seed", range(12))
def test_any_sequence_of_steps(copies, seed):
    rng = random.Random(seed)
    book = Book()
    c = book.cache
    for step in range(150):
        what = rng.choice(["grow"] * 6 + ["fork", "reorder", "reorder", "release", "compact", "back"])
        known = sorted(book.said)
        if what in ("grow", "back"):
            some = rng.sample(known, min(len(known), rng.randint(0, 4))) + ([max(known, default=0) + 1] if rng.random() < 0.2 else [])
            counts = [rng.randint(0, 6) for _ in some]
            before, lists = dict(c.lengths), {r: list(p) for r, p in c.pages.items()}
            try:
                if what == "grow":
                    book.grow(some, counts)
                else:
                    c.grow(some, counts)
                    c.take_back(some, counts)
                    # Counts of zero of a request that was not there leave none behind.
            except RuntimeError:  # not enough pages: all as it was
                assert c.lengths == before and c.pages == lists
        elif what == "fork" and known and len(known) < 8:
            a, b = rng.choice(known), known[-1] + 1
            c.fork(a, b)
            book.said[b] = list(book.said[a])
        elif what == "reorder" and known:
            some = rng.sample(known, rng.randint(1, len(known)))
            parents = [rng.randrange(-1, len(some)) for _ in some]
            c.reorder(some, parents)
            now = {r: list(book.said[some[p]]) for r, p in zip(some, parents) if p >= 0}
            for r in some:
                del book.said[r]
            book.said.update(now)
        elif what == "release" and known:
            r = rng.choice(known)
            c.release(r)
            del book.said[r]
        elif what == "compact":
            used = c.compact()
            assert {p for pages in c.pages.values() for p in pages} == set(range(used))
        # A request that stands at nothing may or may not be listed.
        book.said = {r: t for r, t in book.said.items() if t or r in c.lengths}
        for r in list(c.lengths):
            if not c.lengths[r]:
                book.said.setdefault(r, [])
                c.pages.setdefault(r, [])
        book.check()
    assert copies


def test_only_a_shared_page_that_is_written_is_copied(copies):
    book = Book(page=4)
    c = book.cache
    book.grow([0], [10])
    c.fork(0, 1)
    c.fork(0, 2)
    book.said[1], book.said[2] = list(book.said[0]), list(book.said[0])
    assert len(c.free) == 40 - 3 and not copies
    book.grow([1, 0, 2], [1, 1, 1])  # three requests, one page: two copies
    book.check()
    assert len(copies) == 1 and len(copies[0]) == 2 and {s for s, _ in copies[0]} == {c.pages[2][2]}
    book.grow([1, 0, 2], [1, 1, 1])
    assert len(copies) == 1
    c.fork(1, 3)  # full pages are only read
    book.said[3] = list(book.said[1])
    book.grow([3], [5])
    book.check()
    assert len(copies) == 1
    for r in range(4):
        c.release(r)
    assert sorted(c.free) == list(range(40)) and not c.shares


def test_refusals(copies):
    book = Book(pages=4)
    c = book.cache
    book.grow([0, 1], [6, 3])
    before = (list(c.free), dict(c.lengths), {r: list(p) for r, p in c.pages.items()})
    for call in (lambda: c.fork(5, 6), lambda: c.fork(0, 1), lambda: c.reorder([0, 0], [0, 0]), lambda: c.reorder([0], [1]),
                 lambda: c.reorder([0, 1], [0]), lambda: c.reorder([0, 7], [1, 0]), lambda: c.resize(2)):
        with pytest.raises(ValueError):
            call()
    assert (c.free, c.lengths, c.pages) == before
    for dtype in (torch.float32, torch.uint8):
        with pytest.raises(ValueError):
            PagedCache(1, 2, 1, 16, 64, device="cpu", dtype=dtype)
    with pytest.raises(ValueError):
        PagedCache(1, 2, 1, 8, 64, device="cpu", dtype=torch.int8)


def test_a_copy_that_fails_leaves_the_cache_as_it_was(monkeypatch):
    book = Book()
    c = book.cache
    book.grow([0], [5])
    c.fork(0, 1)
    before = (list(c.free), dict(c.lengths), {r: list(p) for r, p in c.pages.items()}, dict(c.shares))

    def fail(*a):
        raise RuntimeError("no")

    monkeypatch.setattr(ops, "paged_copy", fail)
    with pytest.raises(RuntimeError):
        c.grow([0, 1], [1, 1])
    assert (c.free, c.lengths, c.pages, c.shares) == before


def test_resize(copies):
    book = Book(pages=12)
    c = book.cache
    book.grow([0, 1, 2], [9, 5, 7])
    c.release(1)
    del book.said[1]
    c.fork(2, 3)
    book.said[3] = list(book.said[2])
    c.resize(5)
    assert c.k.shape[1] == c.v.shape[1] == 5 and not c.free
    book.check()
    c.resize(30)
    assert len(c.free) == 25
    book.grow([3, 2], [9, 1])
    book.check()
    eight = PagedCache(2, 9, 3, 32, 64, device="cpu", dtype=torch.int8)
    assert eight.k_scales.shape == (2, 9, 3, 2) and len(eight.arrays()) == 4 and set(eight.scales(1)) == {"k_scales", "v_scales"}
    eight.resize(4)
    assert eight.k_scales.shape == (2, 4, 3, 2)


# ---------------------------------------------------------------- beam search around a model of a few lines


class Chain:
    """Next-token logits from a table by the last two tokens, read back from the cache's own slots."""

    def __init__(self, vocab, seed=0, end_bias=0.0):
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randn(vocab, vocab, vocab, generator=g) * 2
        self.table[..., 0] += end_bias
        self.vocab = vocab

    def step(self, cache, names, parts):
        assert all(parts)
        counts = [len(p) for p in parts]
        cache.grow(names, counts)
        rows = []
        for n, p in zip(names, parts):
            L, size = cache.lengths[n], cache.page_size
            for i, t in enumerate(p):
                at = L - len(p) + i
                cache.k[0, cache.pages[n][at // size], 0, at % size, 0] = t
            seen = [int(cache.k[0, cache.pages[n][t // size], 0, t % size, 0]) for t in range(L)]
            rows += [self.table[seen[t - 1] if t else 0, seen[t]] for t in range(L - len(p), L)]
        return torch.stack(rows)

    def logits(self, seen):
        return self.table[seen[-2] if len(seen) > 1 else 0, seen[-1]]


def plain_select(logits, scores, count=None, finished=None, end=-1):
    from tests.test_gpu_beams import reference
    best, parent, token = reference(logits, scores, scores.shape[1] if count is None else count, finished, end)
    return ops.BeamChoice(best.float(), parent, token)


def plain_search(model, prompt, beams, new_tokens, end):
    live = [Hypothesis([], 0.0)]
    for _ in range(new_tokens):
        every = []
        for h in live:
            if h.ended:
                every.append(h)
                continue
            p = torch.log_softmax(model.logits(prompt + h.tokens).double(), -1) + float(torch.tensor(h.score, dtype=torch.float32))
            every += [Hypothesis(h.tokens + [t], float(p[t]), t == end) for t in range(model.vocab)]
        live = sorted(every, key=lambda h: -h.score)[:beams]
        live = [Hypothesis(h.tokens, float(torch.tensor(h.score, dtype=torch.float32)), h.ended) for h in live]
    return live


@pytest.mark.parametrize("beams,new,end,bias,page,chunk", [(1, 5, None, 0, 4, 3), (4, 9, None, 0, 4, 256), (3, 12, 0, 1.5, 4, 2),
                                                          (8, 6, 0, 4.0, 8, 5), (30, 4, None, 0, 4, 4), (5, 0, None, 0, 4, 4)])
def test_beam_search_finds_what_a_plain_search_finds(copies, monkeypatch, beams, new, end, bias, page, chunk):
    monkeypatch.setattr(ops, "beam_select", plain_select)
    model = Chain(11, seed=beams, end_bias=bias)
    prompts = [[1, 2, 3, 4, 5], [7], [3] * 9]
    cache = PagedCache(1, 200, 1, page, 64, device="cpu")
    cache.grow([2], [6])  # somebody else's
    before = dict(cache.lengths), {r: list(p) for r, p in cache.pages.items()}
    got = beam_search(model, cache, prompts, beams, new, end=end, chunk=chunk)
    assert (cache.lengths, cache.pages) == before and len(cache.free) == 200 - len(cache.pages[2]) and not cache.shares
    for prompt, found in zip(prompts, got):
        want = plain_search(model, prompt, beams, new, end) if new else []
        assert [h.tokens for h in found] == [h.tokens for h in want]
        assert [h.ended for h in found] == [h.ended for h in want]
        assert all(abs(a.score - b.score) < 1e-4 for a, b in zip(found, want))


def test_beam_search_gives_its_pages_back(copies, monkeypatch):
    monkeypatch.setattr(ops, "beam_select", plain_select)
    model = Chain(11)
    cache = PagedCache(1, 9, 1, 4, 64, device="cpu")
    with pytest.raises(RuntimeError):
        beam_search(model, cache, [[1, 2, 3]], 6, 20)
    assert len(cache.free) == 9 and not cache.pages and not cache.lengths and not cache.shares
    for kw in (dict(beams=0), dict(beams=65), dict(chunk=0), dict(new_tokens=-1), dict(prompts=[[1], []])):
        args = dict(prompts=[[1]], beams=2, new_tokens=2, chunk=4) | kw
        with pytest.raises(ValueError):
            beam_search(model, cache, **args)
    assert beam_search(model, cache, [], 3, 4) == []


def test_beam_search_refuses_logits_that_are_no_distribution(copies, monkeypatch):
    """As serve does: an error, not an empty answer; its pages are free again."""
    from trifuse_b200 import TriFuseError
    monkeypatch.setattr(ops, "beam_select", plain_select)
    for bad in ("at once", "later"):
        model = Chain(11)
        if bad == "at once":
            model.table[:] = float("nan")
        else:
            model.table[3:, 3:] = float("inf")
        cache = PagedCache(1, 90, 1, 4, 64, device="cpu")
        with pytest.raises(TriFuseError, match="no distribution"):
            beam_search(model, cache, [[1, 2], [5, 7]], 3, 20)
        assert len(cache.free) == 90 and not cache.pages and not cache.lengths
