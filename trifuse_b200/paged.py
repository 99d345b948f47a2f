"""Serving over a paged key/value cache: prompt chunks, decode steps and log
probabilities in one loop, and beam search.

``PagedCache`` owns a model's pages, in 16 or 8 bits, and lends them to
requests, which may share them; ``PagedOLMoE`` runs OLMoE steps over it from the
operators in ``trifuse_b200.ops``: every step takes any mix of prompt chunks and
single tokens (one attention plan for all layers).  ``serve`` reports each
token's log probability, entropy, rank and alternatives; ``beam_search`` keeps
the most probable continuations of each prompt.

    python -m trifuse_b200.paged                            # a small synthetic model
    python -m trifuse_b200.paged --cache int8 --beams 4     # beam search over an 8-bit cache
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
    page_size, head_dim] and the requests' page lists.  dtype: float16, or
    int8 or float8_e4m3fn with a scale for each 16 tokens of a head.

    Requests may share pages (``fork``, ``reorder``); a page that is shared and
    not full is copied for the request that is about to write to it (``grow``)."""

    def __init__(self, layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda",
                 dtype=torch.float16):
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.k_scales = self.v_scales = None
        if dtype in (torch.int8, torch.float8_e4m3fn):
            if page_size % ops.SCALE_TOKENS:
                raise ValueError("paged cache: pages of an 8-bit cache hold a multiple of 16 tokens")
            shape = (layers, pages, kv_heads, page_size // ops.SCALE_TOKENS)
            self.k_scales = torch.empty(shape, dtype=torch.float32, device=device)
            self.v_scales = torch.empty(shape, dtype=torch.float32, device=device)
        elif dtype != torch.float16:
            raise ValueError("paged cache: float16, int8 or float8_e4m3fn")
        self.page_size = page_size
        self.free = list(range(pages - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}
        self.lengths: dict[int, int] = {}
        self.shares: dict[int, int] = {}  # requests that list a page, where they are several

    def arrays(self):
        """The tensors [layers, pages, ...] that hold the cache."""
        return [t for t in (self.k, self.v, self.k_scales, self.v_scales) if t is not None]

    def scales(self, layer: int) -> dict:
        """Arguments of the paged operators beside a layer's pages."""
        if self.k_scales is None:
            return {}
        return dict(k_scales=self.k_scales[layer], v_scales=self.v_scales[layer])

    def _own(self, request, count):
        """Whether the request's last page has to become its own before `count`
        tokens are written."""
        length = self.lengths.get(request, 0)
        return count > 0 and length % self.page_size > 0 and self.pages[request][length // self.page_size] in self.shares

    def grow(self, requests, counts):
        """Room for counts[i] more tokens of requests[i], each listed once; all
        or nothing."""
        if len(requests) != len(counts) or any(n < 0 for n in counts):
            raise ValueError("paged cache: a count of new tokens, not negative, for each request")
        if len(set(requests)) != len(requests):  # its rows would be given the same slots twice
            raise ValueError("paged cache: a request is listed twice")
        need = [max(0, -(-(self.lengths.get(r, 0) + n) // self.page_size) - len(self.pages.get(r, ())))
                for r, n in zip(requests, counts)]
        # The last of those that share a page keeps it.
        left = {}
        apart = []
        for r, n in zip(requests, counts):
            if self._own(r, n):
                page = self.pages[r][self.lengths[r] // self.page_size]
                if left.setdefault(page, self.shares[page]) > 1:
                    left[page] -= 1
                    apart.append(r)
        if sum(need) + len(apart) > len(self.free):
            raise RuntimeError(f"paged cache: {sum(need) + len(apart)} pages needed, {len(self.free)} free")
        if apart:
            at = [self.lengths[r] // self.page_size for r in apart]
            dst = self.free[: -len(apart) - 1: -1]
            ops.paged_copy(self.arrays(), [self.pages[r][i] for r, i in zip(apart, at)], dst)
            del self.free[-len(apart):]
            for r, i, page in zip(apart, at, dst):
                self._drop(self.pages[r][i])
                self.pages[r][i] = page
        for r, n, count in zip(requests, need, counts):
            self.pages.setdefault(r, []).extend(self.free.pop() for _ in range(n))
            self.lengths[r] = self.lengths.get(r, 0) + count

    def take_back(self, requests, counts):
        """Undoes the last grow of the same requests and counts (pages that it
        copied stay their requests' own).  What was written to an 8-bit cache
        meanwhile is not undone in blocks that hold earlier tokens: a scale that
        rose stays, with the earlier codes rounded to it, and one that a NaN or
        an infinity made NaN does too, so these up to 15 tokens are lost until
        they are appended again, from the block's first on."""
        for r, count in reversed(list(zip(requests, counts))):
            left = self.lengths[r] - count
            keep = -(-left // self.page_size)
            pages = self.pages[r]
            self._give_back(pages[keep:])
            del pages[keep:]
            self.lengths[r] = left
            if left == 0:
                self.release(r)

    def _drop(self, page):
        """One request fewer lists the page; True when none does."""
        if page not in self.shares:
            return True
        self.shares[page] -= 1
        if self.shares[page] == 1:
            del self.shares[page]
        return False

    def _give_back(self, pages):
        self.free.extend(p for p in reversed(pages) if self._drop(p))

    def release(self, request: int):
        pages = self.pages.pop(request, [])
        self.free.extend(p for p in pages if self._drop(p))
        self.lengths.pop(request, None)

    def fork(self, request: int, other: int):
        """`other`, a new request, begins where `request` stands and shares its
        pages."""
        if request not in self.lengths:
            raise ValueError("paged cache: no such request")
        if other in self.lengths or other in self.pages:
            raise ValueError("paged cache: the new request is there already")
        self.pages[other] = list(self.pages[request])
        self.lengths[other] = self.lengths[request]
        for p in self.pages[other]:
            self.shares[p] = self.shares.get(p, 1) + 1

    def reorder(self, requests, parents):
        """requests[i] goes on from where requests[parents[i]] stands (below 0:
        it ends); requests that nobody goes on from give their pages back."""
        if len(requests) != len(parents) or any(p >= len(requests) for p in parents):
            raise ValueError("paged cache: a parent among the requests for each of them")
        if len(set(requests)) != len(requests):
            raise ValueError("paged cache: a request is listed twice")
        if any(p >= 0 and requests[p] not in self.lengths for p in parents):
            raise ValueError("paged cache: no such request")
        now = [(list(self.pages[requests[p]]), self.lengths[requests[p]]) if p >= 0 else None for p in parents]
        for state in now:
            for page in state[0] if state else ():
                self.shares[page] = self.shares.get(page, 1) + 1
        for r in requests:
            self.release(r)
        for r, state in zip(requests, now):
            if state:
                self.pages[r], self.lengths[r] = state

    def compact(self) -> int:
        """Moves the pages in use to the front of the cache; returns how many
        there are."""
        used = sorted({p for pages in self.pages.values() for p in pages})
        to = dict(zip(used, used))
        holes = sorted(set(range(len(used))) - set(used))
        moved = [p for p in used if p >= len(used)]
        to.update(zip(moved, holes))
        if moved:
            ops.paged_copy(self.arrays(), moved, holes)
        for pages in self.pages.values():
            pages[:] = [to[p] for p in pages]
        self.shares = {to[p]: n for p, n in self.shares.items()}
        self.free = list(range(self.k.shape[1] - 1, len(used) - 1, -1))
        return len(used)

    def resize(self, pages: int):
        """Another number of pages, no fewer than are in use.  Where memory does
        not suffice for all arrays, each keeps the smaller number."""
        used = len({p for lists in self.pages.values() for p in lists})
        if pages < used:
            raise ValueError(f"paged cache: {used} pages are in use")
        used = self.compact()
        names = [n for n in ("k", "v", "k_scales", "v_scales") if getattr(self, n) is not None]
        try:
            for name in names:  # one after the other: each takes the old one's place
                old = getattr(self, name)
                new = old.new_empty((old.shape[0], pages, *old.shape[2:]))
                new[:, :used] = old[:, :used]
                setattr(self, name, new)
        finally:
            pages = min(getattr(self, n).shape[1] for n in names)
            for name in names:
                if getattr(self, name).shape[1] > pages:
                    setattr(self, name, getattr(self, name)[:, :pages])
            self.free = list(range(pages - 1, used - 1, -1))

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
                                 eps=cfg.rms_eps, rope_theta=cfg.rope_theta, **cache.scales(l))
            o = ops.paged_attention(q, cache.k[l], cache.v[l], table, plan, **cache.scales(l))
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


@dataclass
class Hypothesis:
    """Tokens that beam search generated after a prompt, and their log probability."""
    tokens: list
    score: float
    ended: bool = False


def beam_search(model: PagedOLMoE, cache: PagedCache, prompts, beams: int, new_tokens: int, end: int | None = None,
                chunk: int = 256) -> list[list[Hypothesis]]:
    """Up to `beams` most probable continuations of each prompt, best first, of
    `new_tokens` tokens or until the token `end`: at each step the best beams *
    (beams * vocabulary) continuations go on.  A prompt is read once (up to
    `chunk` of its tokens a step) and its pages are shared by its beams.  The
    cache may hold other requests; the pages of these are free again when the
    call ends, also by an exception."""
    if chunk < 1 or not 1 <= beams <= 64 or new_tokens < 0:
        raise ValueError("beam_search: chunk and beams (at most 64) are positive, new_tokens is not negative")
    if any(not p for p in prompts):
        raise ValueError("beam_search: a prompt is empty")
    R = len(prompts)
    unused = (n for n in itertools.count() if n not in cache.lengths and n not in cache.pages)
    names = [list(itertools.islice(unused, beams)) for _ in range(R)]
    found = [[] for _ in range(R)]
    if R == 0 or new_tokens == 0:
        return found
    try:
        # The prompts: the first beam reads, the others join it.
        logits, fed, active = [None] * R, 0, list(range(R))
        while active:
            parts = [prompts[r][fed: fed + chunk] for r in active]
            out = model.step(cache, [names[r][0] for r in active], parts)
            row = 0
            for r, p in zip(active, parts):
                row += len(p)
                if fed + chunk >= len(prompts[r]):
                    logits[r] = out[row - 1].clone()  # the rest of the step's logits may go
            fed += chunk
            active = [r for r in active if len(prompts[r]) > fed]
        got = ops.beam_select(torch.stack(logits)[:, None], torch.zeros(R, 1, device=cache.k.device), beams)
        ended = [[False] * beams for _ in range(R)]
        for step in range(new_tokens):
            parents, tokens, scores = got.parent.tolist(), got.token.tolist(), got.score.tolist()
            for r in range(R):
                before = found[r] or [Hypothesis([], 0.0)]
                if step == 0:
                    for b, p in enumerate(parents[r][1:], 1):
                        if p >= 0:
                            cache.fork(names[r][0], names[r][b])
                else:
                    cache.reorder(names[r], parents[r])
                found[r] = [Hypothesis(before[p].tokens + [t] * (not before[p].ended), s,
                                       before[p].ended or t == end) if p >= 0 else None
                            for p, t, s in zip(parents[r], tokens[r], scores[r])]
                if not any(found[r]):  # as serve refuses such a row
                    raise TriFuseError(9, "beam_search: logits that are no distribution give no continuation")
                ended[r] = [h is None or h.ended for h in found[r]]
                for b in range(beams):
                    if ended[r][b]:  # its tokens are all that is left of it
                        cache.release(names[r][b])
                        cache.lengths[names[r][b]], cache.pages[names[r][b]] = 0, []
            if step + 1 == new_tokens or all(map(all, ended)):
                break
            live = [(r, b) for r in range(R) for b in range(beams) if not ended[r][b]]
            out = model.step(cache, [names[r][b] for r, b in live], [[found[r][b].tokens[-1]] for r, b in live])
            finished = None
            if len(live) < R * beams:  # rows of ended beams are not read
                at = torch.tensor([r * beams + b for r, b in live]).to(out.device)
                out = out.new_empty((R * beams, out.shape[1])).index_copy_(0, at, out)
                finished = torch.tensor(ended).to(out.device)
            got = ops.beam_select(out.view(R, beams, -1), got.score, beams, finished=finished,
                                  end=-1 if end is None else end)
    finally:
        for group in names:
            for n in group:
                cache.release(n)
    return [[h for h in hs if h is not None] for hs in found]


CACHES = {"f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def main(argv=None):
    from .quant import synthetic_olmoe
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--new", type=int, default=8)
    ap.add_argument("--cache", choices=CACHES, default="f16")
    ap.add_argument("--beams", type=int, default=0, help="beam search with that many beams a request")
    a = ap.parse_args(argv)
    cfg = Config(layers=a.layers, vocab=4096)
    model = PagedOLMoE(cfg, synthetic_olmoe(cfg, seed=1, device="cuda"))
    longest = a.prompt + 37 * a.requests + a.new
    each = -(-longest // 16) + max(a.beams - 1, 0) * (a.new // 16 + 2)  # beams share the prompt's pages
    cache = PagedCache(cfg.layers, a.requests * each, cfg.kv_heads, 16, cfg.head_dim, dtype=CACHES[a.cache])
    g = torch.Generator().manual_seed(2)
    reqs = [Request(torch.randint(0, cfg.vocab, (a.prompt + 37 * i,), generator=g).tolist(), a.new)
            for i in range(a.requests)]
    if a.beams:
        for i, found in enumerate(beam_search(model, cache, [r.prompt for r in reqs], a.beams, a.new)):
            for h in found:
                print(f"request {i}: log probability {h.score:.3f}: {h.tokens}")
    else:
        for i, r in enumerate(serve(model, cache, reqs)):
            mean = sum(r.prompt_logprobs) / max(len(r.prompt_logprobs), 1)
            print(f"request {i}: prompt {len(r.prompt)} tokens, mean log probability {mean:.3f}; generated {r.tokens} "
                  f"with {[round(x, 3) for x in r.logprobs]}")
    if ops.device_error():
        raise RuntimeError("a device-side wait expired")


if __name__ == "__main__":
    main()
