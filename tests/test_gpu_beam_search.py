"""OLMoE over 8-bit caches, and beam search over any of them: append, attention, selection and page copies as they run
together."""
import numpy as np
import pytest
import torch

from tests.test_gpu_model import oracle_weights, tiny_cfg
from tests.test_gpu_paged_model import exact

pytestmark = pytest.mark.gpu

KINDS = {"f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def model():
    from trifuse_b200.paged import PagedOLMoE
    from trifuse_b200.quant import synthetic_olmoe
    cfg = tiny_cfg(torch.float16)
    w = synthetic_olmoe(cfg, seed=7, device="cuda")
    return cfg, PagedOLMoE(cfg, w), oracle_weights(w, cfg)


def cache_for(cfg, kind, pages=80, page=16):
    from trifuse_b200.paged import PagedCache
    c = PagedCache(cfg.layers, pages, cfg.kv_heads, page, cfg.head_dim, dtype=KINDS[kind])
    for t in c.arrays():  # a former owner's: NaN codes and scales where there are any
        t.view(torch.uint8).fill_(0x7f)
    return c


def copying(cache):
    """The cache with pages of its own for every request instead of shared ones."""
    from trifuse_b200 import ops

    class Copying(type(cache)):
        def fork(self, request, other):
            super().fork(request, other)
            self.apart(other)

        def apart(self, request):
            for i, p in enumerate(self.pages[request]):
                if p in self.shares:
                    new = self.free.pop()
                    ops.paged_copy(self.arrays(), [p], [new])
                    self._drop(p)
                    self.pages[request][i] = new

        def reorder(self, requests, parents):
            super().reorder(requests, parents)
            for r in requests:
                if r in self.pages:
                    self.apart(r)

    cache.__class__ = Copying
    return cache


@pytest.mark.parametrize("kind,limit", [("f16", 0.02), ("int8", 0.05), ("e4m3", 0.15)])
def test_chunks_and_decode_steps(model, kind, limit):
    """The last rows' logits against a forward in 64 bits.  A value of the cache is off by 1/254 of its block's largest
    at most, 0.8 per cent rms of a normal block (int8), or by 2^-4 of itself, 2.5 per cent rms (e4m3).  Keys and
    values add up, and a layer's attention is one of three terms of the residual: the logits' norm moves by a few of
    these."""
    cfg, m, ow = model
    cache = cache_for(cfg, kind)
    rng = np.random.default_rng(0)
    ids = {r: rng.integers(0, cfg.vocab, size=45).tolist() for r in range(3)}
    done = {r: 0 for r in range(3)}
    worst = 0.0
    for counts in ({0: 20, 1: 7, 2: 33}, {0: 1, 1: 17, 2: 1}, {0: 1, 1: 1, 2: 1}, {0: 5, 2: 1}):
        parts = [ids[r][done[r]: done[r] + n] for r, n in counts.items()]
        out = m.step(cache, list(counts), parts)
        row = -1
        for r, p in zip(counts, parts):
            row += len(p)
            done[r] += len(p)
            want = exact(ids[r][: done[r]], cfg, ow)
            got = out[row].double().cpu().numpy()
            assert np.isfinite(got).all()
            worst = max(worst, np.linalg.norm(got - want) / np.linalg.norm(want))
    assert worst <= limit, worst


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32])
def test_shared_pages_give_the_bits_of_pages_of_ones_own(model, kind, page):
    from trifuse_b200 import ops
    from trifuse_b200.paged import beam_search
    cfg, m, _ = model
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.vocab, size=n).tolist() for n in (37, 5, 16)]
    shared, own = cache_for(cfg, kind, page=page), copying(cache_for(cfg, kind, page=page))
    a = beam_search(m, shared, prompts, 4, 21, end=3, chunk=20)
    b = beam_search(m, own, prompts, 4, 21, end=3, chunk=20)
    assert ops.device_error() == 0
    assert [[(h.tokens, h.score) for h in hs] for hs in a] == [[(h.tokens, h.score) for h in hs] for hs in b]
    assert len(shared.free) == len(own.free) == 80
    for hs in a:
        assert len(hs) == 4 and all(x.score >= y.score for x, y in zip(hs, hs[1:]))
        assert all(len(h.tokens) == 21 or h.tokens[-1] == 3 for h in hs) and len({tuple(h.tokens) for h in hs}) == 4


def test_scores_are_those_of_the_tokens(model):
    """A found continuation read as a prompt has the log probabilities that add up to its score: each is off by the
    f16 rounding of its logits and what lies between a chunk's sums and a single token's, some 2^-11 of logits below
    16, twice."""
    from trifuse_b200.paged import Request, beam_search, serve
    cfg, m, _ = model
    prompt = np.random.default_rng(5).integers(0, cfg.vocab, size=23).tolist()
    n = 12
    found = beam_search(m, cache_for(cfg, "f16"), [prompt], 5, n)[0]
    reqs = serve(m, cache_for(cfg, "f16"), [Request(prompt + h.tokens, 0) for h in found])
    for h, r in zip(found, reqs):
        assert abs(sum(r.prompt_logprobs[len(prompt) - 1:]) - h.score) <= n * 2 * 16 * 2.0 ** -11
    greedy = serve(m, cache_for(cfg, "f16"), [Request(prompt, n)])[0]
    assert found[0].score >= sum(greedy.logprobs) - n * 2 * 16 * 2.0 ** -11
    one = beam_search(m, cache_for(cfg, "f16"), [prompt], 1, n)[0][0]
    assert one.tokens == greedy.tokens and abs(one.score - sum(greedy.logprobs)) <= 1e-4


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_serve_over_8_bits(model, kind):
    """The serving loop with prompts that are read in chunks beside others that generate, after a compaction too."""
    from trifuse_b200.paged import Request, serve
    cfg, m, _ = model
    rng = np.random.default_rng(6)
    cache = cache_for(cfg, kind)
    cache.grow([100, 101], [40, 70])
    cache.release(100)
    reqs = [Request(rng.integers(0, cfg.vocab, size=k).tolist(), 6) for k in (30, 3, 50)]
    serve(m, cache, reqs, chunk=16)
    cache.compact()
    again = [Request(r.prompt, 6) for r in reqs]
    serve(m, cache, again, chunk=16)
    for a, b in zip(reqs, again):
        assert a.tokens == b.tokens and a.logprobs == b.logprobs and all(np.isfinite(a.prompt_logprobs))


def test_resize_keeps_what_requests_hold(model):
    cfg, m, _ = model
    rng = np.random.default_rng(8)
    logits = []
    for move in (False, True):
        cache = cache_for(cfg, "e4m3")
        cache.grow([7], [100])
        m.step(cache, [1, 2], [list(range(30)), list(range(50))])
        cache.release(7)
        if move:
            cache.resize(12)
        logits.append(m.step(cache, [2, 1], [[5], [6, 7]]))
    assert torch.equal(*logits)
    assert cache.k.shape[1] == 12


def test_command(capsys):
    from trifuse_b200.paged import main
    main(["--layers", "1", "--requests", "2", "--prompt", "40", "--new", "3", "--cache", "int8", "--beams", "3"])
    assert capsys.readouterr().out.count("log probability") == 6
    main(["--layers", "1", "--requests", "2", "--prompt", "40", "--new", "3", "--cache", "e4m3"])
    assert capsys.readouterr().out.count("generated") == 2
