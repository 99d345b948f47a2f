"""OLMoE over a paged cache: chunks beside decode steps against a forward in 64 bits (where the oracle, which rounds
to the activation dtype at more places, sets how far off a forward in that dtype may be), and the serving loop's log
probabilities against the logits they come from."""
import math

import numpy as np
import pytest
import torch

import oracle
from tests.gpu_util import host
from tests.test_gpu_model import oracle_weights, tiny_cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["f16", "bf16"])
def paged(request):
    from trifuse_b200.paged import PagedOLMoE
    from trifuse_b200.quant import synthetic_olmoe
    act = request.param
    cfg = tiny_cfg(torch.float16 if act == "f16" else torch.bfloat16)
    w = synthetic_olmoe(cfg, seed=7, device="cuda")
    ocfg = oracle.OLMoEConfig(layers=cfg.layers, hidden=cfg.hidden, heads=cfg.heads, head_dim=cfg.head_dim,
                              intermediate=cfg.intermediate, vocab=cfg.vocab, experts=cfg.experts, top_k=cfg.top_k,
                              capacity=64, act=act)
    return cfg, PagedOLMoE(cfg, w), oracle_weights(w, cfg), ocfg, act


def cache_for(cfg, pages=24, page=16):
    from trifuse_b200.paged import PagedCache
    return PagedCache(cfg.layers, pages, cfg.kv_heads, page, cfg.head_dim)


def reference(ids, cfg, ow, ocfg):
    """The last row's logits of the whole prefix."""
    caches = [[np.zeros((cfg.heads, 64, cfg.head_dim), np.float32) for _ in range(cfg.layers)] for _ in range(2)]
    return oracle.model_forward(np.asarray(ids), ow, ocfg, caches[0], caches[1], 0)


def exact(ids, cfg, ow):
    """The last row's logits in 64 bits, from the same quantized weights without any rounding on the way."""
    deq = lambda w: oracle.dequantize(*w).astype(np.float64)  # noqa: E731
    rms = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.rms_eps) * np.asarray(w, np.float64)  # noqa: E731
    T, H, D = len(ids), cfg.heads, cfg.head_dim
    h = deq(ow["embed"])[np.asarray(ids)]
    angle = np.arange(T)[:, None, None] * cfg.rope_theta ** (-2.0 * np.arange(D // 2) / D)
    turn = lambda x: np.concatenate([x[..., : D // 2] * np.cos(angle) - x[..., D // 2:] * np.sin(angle),  # noqa: E731
                                     x[..., : D // 2] * np.sin(angle) + x[..., D // 2:] * np.cos(angle)], -1)
    for w in ow["layers"]:
        x = rms(h, w["input_norm"])
        q = turn(rms(x @ deq(w["q"]).T, w["q_norm"]).reshape(T, H, D))
        k = turn(rms(x @ deq(w["k"]).T, w["k_norm"]).reshape(T, H, D))
        v = (x @ deq(w["v"]).T).reshape(T, H, D)
        s = np.einsum("nhd,khd->hnk", q, k) / math.sqrt(D) + np.where(np.tri(T, dtype=bool), 0, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        h = h + np.einsum("hnk,khd->nhd", p, v).reshape(T, -1) @ deq(w["o"]).T
        x = rms(h, w["post_norm"])
        r = x @ deq(w["router"]).T
        g = np.exp(r - r.max(-1, keepdims=True))
        g /= g.sum(-1, keepdims=True)
        gate, up, down = (deq(w["experts"][n]) for n in ("gate", "up", "down"))
        for t in range(T):
            for e in np.argsort(-r[t], kind="stable")[: cfg.top_k]:
                a = gate[e] @ x[t]
                h[t] = h[t] + g[t, e] * (down[e] @ (a / (1 + np.exp(-a)) * (up[e] @ x[t])))
    return rms(h[-1], ow["final_norm"]) @ deq(ow["lm_head"]).T


def test_mixed_steps_are_as_near_as_the_oracle(paged):
    """Three requests, a step of chunks, a step mixing chunks and single tokens, a step of single tokens: over the
    last rows of all parts, the logits are no further from 64 bits than the oracle's forward of the whole prefix in
    the same dtype, but for a quarter (other sums of the same roundings)."""
    cfg, model, ow, ocfg, act = paged
    cache = cache_for(cfg)
    rng = np.random.default_rng(0)
    ids = {r: rng.integers(0, cfg.vocab, size=40).tolist() for r in range(3)}
    done = {r: 0 for r in range(3)}
    ours, theirs = [], []
    for part in ({0: 17, 1: 1, 2: 20}, {0: 1, 2: 1, 1: 13}, {1: 1, 0: 1, 2: 1}, {2: 9}):
        reqs = list(part)
        logits = host(model.step(cache, reqs, [ids[r][done[r]: done[r] + part[r]] for r in reqs]))
        row = 0
        for r in reqs:
            done[r] += part[r]
            row += part[r]
            want = exact(ids[r][: done[r]], cfg, ow)
            ours.append(np.abs(logits[row - 1] - want).mean())
            theirs.append(np.abs(reference(ids[r][: done[r]], cfg, ow, ocfg) - want).mean())
    assert np.mean(ours) <= 1.25 * np.mean(theirs), (ours, theirs)


def test_serve_reports_log_probabilities(paged):
    """Chunked serving gives what one forward of prompt and answer gives, and leaves every page free."""
    from trifuse_b200.paged import Request, serve
    cfg, model, *_, act = paged
    cache = cache_for(cfg)
    rng = np.random.default_rng(3)
    reqs = [Request(rng.integers(0, cfg.vocab, size=n).tolist(), k) for n, k in ((23, 4), (1, 6), (9, 0), (40, 1))]
    serve(model, cache, reqs, chunk=8, top=3)
    assert sorted(cache.free) == list(range(24)) and not cache.pages
    for r, new in zip(reqs, (4, 6, 0, 1)):
        assert len(r.tokens) == new == len(r.logprobs) and len(r.prompt_logprobs) == len(r.prompt) - 1
        whole = cache_for(cfg)
        text = r.prompt + r.tokens
        lp = torch.log_softmax(model.step(whole, [0], [text]).double(), -1)
        told = torch.tensor(r.prompt_logprobs + r.logprobs, dtype=torch.float64)
        want = lp[torch.arange(len(text) - 1), torch.tensor(text[1:])].cpu()
        # Both sides round activations throughout the forward (other shapes, other
        # kernels); logits here are below 1, so a few of their units cover it.
        assert (told - want).abs().max() <= (2e-2 if act == "f16" else 8e-2) if len(text) > 1 else True
        for best, alt in zip(r.logprobs, r.alternatives):
            assert len(alt) == 3 and alt[0][1] == best and alt[0][1] >= alt[1][1] >= alt[2][1]


def test_cache_refuses_before_it_grows(paged):
    cfg, model, *_ = paged
    cache = cache_for(cfg, pages=2)
    with pytest.raises(RuntimeError, match="pages needed"):
        model.step(cache, [0, 1], [[1] * 20, [2] * 17])
    assert len(cache.free) == 2 and not cache.pages and not cache.lengths
    assert model.step(cache, [0], [[1] * 20]).shape == (20, cfg.vocab)
