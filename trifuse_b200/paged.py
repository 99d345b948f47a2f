"""Serving over a paged key/value cache: prompt chunks, decode steps and log
probabilities in one loop.

``PagedCache`` owns a model's pages and lends them to requests; ``PagedOLMoE``
runs OLMoE steps over it from the operators in ``trifuse_b200.ops``: every step
takes any mix of prompt chunks and single tokens (one attention plan for all
layers), and ``serve`` reports each token's log probability, entropy, rank and
alternatives.

    python -m trifuse_b200.paged            # a small synthetic model
"""
from __future__ import annotations

import argparse
import itertools
import math
from dataclasses import dataclass, field

import torch
from torch import Tensor

from . import ops
from ._lib import TriFuseError
from .model import Config


class PagedCache:
    """Keys and values of every layer in pages [layers, pages, kv_heads,
    page_size, head_dim] (float16) and the requests' page lists."""

    def __init__(self, layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda"):
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=torch.float16, device=device)
        self.v = torch.empty(shape, dtype=torch.float16, device=device)
        self.page_size = page_size
        self.free = list(range(pages - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}
        self.lengths: dict[int, int] = {}

    def grow(self, requests, counts):
        """Room for counts[i] more tokens of requests[i], each listed once; all
        or nothing."""
        if len(requests) != len(counts) or any(n < 0 for n in counts):
            raise ValueError("paged cache: a count of new tokens, not negative, for each request")
        if len(set(requests)) != len(requests):  # its rows would be given the same slots twice
            raise ValueError("paged cache: a request is listed twice")
        need = [max(0, -(-(self.lengths.get(r, 0) + n) // self.page_size) - len(self.pages.get(r, ())))
                for r, n in zip(requests, counts)]
        if sum(need) > len(self.free):
            raise RuntimeError(f"paged cache: {sum(need)} pages needed, {len(self.free)} free")
        for r, n, count in zip(requests, need, counts):
            self.pages.setdefault(r, []).extend(self.free.pop() for _ in range(n))
            self.lengths[r] = self.lengths.get(r, 0) + count

    def take_back(self, requests, counts):
        """Undoes the last grow of the same requests and counts."""
        for r, count in reversed(list(zip(requests, counts))):
            left = self.lengths[r] - count
            keep = -(-left // self.page_size)
            pages = self.pages[r]
            self.free.extend(reversed(pages[keep:]))
            del pages[keep:]
            self.lengths[r] = left
            if left == 0:
                self.release(r)

    def release(self, request: int):
        self.free.extend(self.pages.pop(request, ()))
        self.lengths.pop(request, None)

    def table(self, requests) -> Tensor:
        """Page table of the requests, on the cache's device."""
        wide = max((len(self.pages.get(r, ())) for r in requests), default=0)
        rows = [self.pages.get(r, []) + [-1] * (wide - len(self.pages.get(r, ()))) for r in requests]
        return torch.tensor(rows, dtype=torch.int32).reshape(len(rows), wide).to(self.k.device)


class PagedOLMoE:
    """OLMoE over a paged cache; weights by checkpoint name on the device, as
    ``Model`` takes them."""

    def __init__(self, cfg: Config, weights: dict):
        self.cfg = cfg
        aff = lambda p: tuple(weights[f"{p}.{s}"] for s in ("weight", "scales", "biases"))  # noqa: E731
        self.embed, self.lm_head = aff("model.embed_tokens"), aff("lm_head")
        self.final_norm = weights["model.norm.weight"]
        self.layers = []
        for l in range(cfg.layers):
            p = f"model.layers.{l}."
            attn = [aff(f"{p}self_attn.{n}_proj") for n in "qkv"]
            self.layers.append(dict(
                qkv=tuple(torch.cat(parts) for parts in zip(*attn)),  # one projection for q | k | v
                o=aff(f"{p}self_attn.o_proj"), router=aff(f"{p}mlp.gate"),
                experts=[aff(f"{p}mlp.switch_mlp.{n}_proj") for n in ("gate", "up", "down")],
                **{n: weights[f"{p}{w}.weight"] for n, w in (
                    ("input_norm", "input_layernorm"), ("post_norm", "post_attention_layernorm"),
                    ("q_norm", "self_attn.q_norm"), ("k_norm", "self_attn.k_norm"))}))

    def step(self, cache: PagedCache, requests, token_lists) -> Tensor:
        """Feeds token_lists[i] to requests[i] (a chunk of a prompt or one
        token) and returns the logits of every row, [rows, vocab] in the
        activation dtype.  A step that raises leaves the cache's lengths and
        pages as they were."""
        counts = [len(t) for t in token_lists]
        cache.grow(requests, counts)
        try:
            return self._forward(cache, requests, token_lists, counts)
        except BaseException:
            cache.take_back(requests, counts)
            raise

    def _forward(self, cache: PagedCache, requests, token_lists, counts) -> Tensor:
        cfg = self.cfg
        table = cache.table(requests)
        plan = ops.PagedPlan(counts, [cache.lengths[r] for r in requests], cfg.heads, cfg.kv_heads, cfg.head_dim,
                             cache.page_size)
        ids = torch.tensor([t for tokens in token_lists for t in tokens], dtype=torch.int64).to(cache.k.device)
        h = ops.native_affine_embedding(ids, *self.embed, 64, 4, cfg.act)
        for l, w in enumerate(self.layers):
            x = ops.rms_norm(h, w["input_norm"], cfg.rms_eps)
            q = ops.paged_append(ops.native_affine_qmm(x, *w["qkv"], 64, 4), cache.k[l], cache.v[l], table,
                                 plan.positions, plan.requests, cfg.heads, q_norm=w["q_norm"], k_norm=w["k_norm"],
                                 eps=cfg.rms_eps, rope_theta=cfg.rope_theta)
            o = ops.paged_attention(q, cache.k[l], cache.v[l], table, plan)
            h = h + ops.native_affine_qmm(o.flatten(1), *w["o"], 64, 4)
            h = ops.moe(ops.rms_norm(h, w["post_norm"], cfg.rms_eps), h, w["router"], *w["experts"], cfg.top_k)
        return ops.native_affine_qmm(ops.rms_norm(h, self.final_norm, cfg.rms_eps), *self.lm_head, 64, 4)


@dataclass
class Request:
    """A prompt, how many tokens to generate, and what came of it."""
    prompt: list
    new_tokens: int
    tokens: list = field(default_factory=list)          # generated, greedy
    prompt_logprobs: list = field(default_factory=list)  # of prompt[1:]
    logprobs: list = field(default_factory=list)         # of the generated tokens
    alternatives: list = field(default_factory=list)     # [(token, log probability)] beside each generated token


def serve(model: PagedOLMoE, cache: PagedCache, requests: list[Request], chunk: int = 256, top: int = 5):
    """Runs the requests to the end: each step takes up to `chunk` prompt
    tokens of every request still reading and one token of every other.  The
    cache may hold other requests; the pages of these are free again when the
    call ends, also by an exception, and requests that were cut short may be
    passed again: they go on after the tokens that they have.  A request without
    a prompt is left as it is."""
    if chunk < 1:
        raise ValueError("serve: chunk is a positive number of tokens")
    fed = [0] * len(requests)
    active = [i for i, r in enumerate(requests) if r.prompt]
    unused = (n for n in itertools.count() if n not in cache.lengths and n not in cache.pages)
    names = dict(zip(active, unused))  # in the cache
    for i in active:
        requests[i].prompt_logprobs = []
    try:
        while active:
            parts = []
            for i in active:
                known = requests[i].prompt + requests[i].tokens
                parts.append(known[fed[i]: fed[i] + chunk])
                fed[i] += len(parts[-1])
            logits = model.step(cache, [names[i] for i in active], parts)
            # The token that follows each row, where it is known; else none (-1).
            follow = []
            for i, p in zip(active, parts):
                follow += (requests[i].prompt + requests[i].tokens)[fed[i] - len(p) + 1: fed[i] + 1]
                follow += [-1] * (fed[i] >= len(requests[i].prompt) + len(requests[i].tokens))
            got = ops.token_logprobs(logits, torch.tensor(follow, dtype=torch.int64).to(logits.device), top=max(top, 1))
            logprob, best, token = got.logprob.tolist(), got.top_logprob.tolist(), got.top_token.tolist()
            row = 0
            for i, p in zip(list(active), parts):
                r = requests[i]
                last = row + len(p) - 1
                r.prompt_logprobs += logprob[row: row + max(0, min(len(p), len(r.prompt) - 1 - (fed[i] - len(p))))]
                if follow[last] < 0:  # everything known is read: the next token is the first alternative
                    if len(r.tokens) < r.new_tokens:
                        if math.isnan(best[last][0]):  # as Session.generate_greedy refuses such a row
                            raise TriFuseError(9, "serve: logits that are not finite give no next token")
                        r.tokens.append(token[last][0])
                        r.logprobs.append(best[last][0])
                        r.alternatives.append(list(zip(token[last], best[last]))[:top])
                    if len(r.tokens) >= r.new_tokens:
                        active.remove(i)
                        cache.release(names[i])
                row += len(p)
    finally:
        for i in active:
            cache.release(names[i])
    return requests


def main(argv=None):
    from .quant import synthetic_olmoe
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--new", type=int, default=8)
    a = ap.parse_args(argv)
    cfg = Config(layers=a.layers, vocab=4096)
    model = PagedOLMoE(cfg, synthetic_olmoe(cfg, seed=1, device="cuda"))
    longest = a.prompt + 37 * a.requests + a.new
    cache = PagedCache(cfg.layers, a.requests * -(-longest // 16), cfg.kv_heads, 16, cfg.head_dim)
    g = torch.Generator().manual_seed(2)
    reqs = [Request(torch.randint(0, cfg.vocab, (a.prompt + 37 * i,), generator=g).tolist(), a.new)
            for i in range(a.requests)]
    for i, r in enumerate(serve(model, cache, reqs)):
        mean = sum(r.prompt_logprobs) / max(len(r.prompt_logprobs), 1)
        print(f"request {i}: prompt {len(r.prompt)} tokens, mean log probability {mean:.3f}; generated {r.tokens} "
              f"with {[round(x, 3) for x in r.logprobs]}")
    if ops.device_error():
        raise RuntimeError("a device-side wait expired")


if __name__ == "__main__":
    main()
