"""Measured cases of beam search over a paged cache held in 8 bits.

Four operators that such a search runs one after the other.  ``paged_append``
stores the new tokens' keys and values as 8-bit codes with a scale for each
block of 16 tokens and head.  ``paged_attention`` lets the new tokens attend
that cache.  ``beam_select`` picks the best continuations over all beams and
the vocabulary.  ``paged_copy`` gives a forked beam its own copy of pages, and
moves pages together.

``own`` selects between the plain torch form of each operator (False) and the
framework's kernels (True).
"""
import math
import random

import torch

own = False

F16, BF16, F32, INT8, E4M3 = "f16", "bf16", "f32", "int8", "e4m3"
DTYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32, INT8: torch.int8,
          E4M3: torch.float8_e4m3fn}
LARGEST = {INT8: 127.0, E4M3: 448.0}  # code that a block's largest magnitude becomes
BLOCK = 16                            # tokens that share a scale
EPS = 1e-5
THETA = 10000.0
# Cost bounds of a drawn case: what the largest listed cases reach.
MAX_SCORES = 1.1e9   # padded (head, query, key) triples of the plain form
MAX_CACHE = 1.1e9    # bytes of codes that one call sees
MAX_LOGITS = 1.1e8   # bytes of logits
MAX_COPY = 6.5e8     # bytes that one call moves
MAX_VALUES = 4e6     # codes of a cache that is handed out as values


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # One decode step of 64 requests of this model's layer: one new token each, which
        # joins the block of the 15 before it.
        dict(name="append-decode-64", op="append", requests=64, new=1, kv=4096, heads=16, kv_heads=16, head_dim=128,
             page=64, act=BF16, cache=E4M3, norm=True, mix=1),
        # A prefill of 8 prompts of 2048 tokens, the same layer.
        dict(name="append-prefill-16384", op="append", requests=8, new=2048, kv=2048, heads=16, kv_heads=16,
             head_dim=128, page=64, act=BF16, cache=E4M3, norm=True, mix=2),
        # Drafted tokens after short histories: blocks that are begun, joined and left; grouped
        # heads, no norm.
        dict(name="append-int8-24x7", op="append", requests=24, new=7, kv=61, heads=32, kv_heads=8, head_dim=128,
             page=16, act=F16, cache=INT8, norm=False, mix=3),
        # One request's decode step on a short history: nothing but latency.
        dict(name="decode-1x600", op="attention", requests=1, new=1, kv=600, ragged=False, heads=16, kv_heads=16,
             head_dim=128, page=16, act=F16, cache=INT8, mix=4),
        # The decode batch of this repository's benchmark: 64 requests at 4096 tokens.
        dict(name="decode-64x4096", op="attention", requests=64, new=1, kv=4096, ragged=False, heads=16, kv_heads=16,
             head_dim=128, page=64, act=BF16, cache=E4M3, mix=5),
        # A serving batch whose histories differ by a factor of sixteen, grouped heads.
        dict(name="decode-ragged-37", op="attention", requests=37, new=1, kv=32768, ragged=True, heads=32, kv_heads=8,
             head_dim=128, page=16, act=BF16, cache=INT8, mix=6),
        # Prompt chunks and decoding requests mixed in one step, narrow heads, odd lengths.
        dict(name="mixed-12", op="attention", requests=12, new=601, kv=8003, ragged=True, heads=14, kv_heads=2,
             head_dim=64, page=32, act=F16, cache=E4M3, mix=7),
        # A late chunk of a long document: 2048 new tokens after 14336.
        dict(name="chunk-2048-of-16384", op="attention", requests=1, new=2048, kv=16384, ragged=False, heads=32,
             kv_heads=8, head_dim=128, page=128, act=BF16, cache=INT8, mix=8),
        # One request's step with four beams.
        dict(name="beams-1x4", op="beams", requests=1, beams=4, count=4, vocab=50304, act=F32, finished=False),
        # A batch's step with eight beams, some of which have ended.
        dict(name="beams-64x8", op="beams", requests=64, beams=8, count=8, vocab=50304, act=F32, finished=True),
        # Two beams of a request part: the page that both write is copied, in every layer.
        dict(name="copy-fork-3", op="copy", layers=16, pages=96, pairs=3, kv_heads=16, page=16, head_dim=128,
             cache=INT8, mix=9),
        # A cache is moved together before it shrinks.
        dict(name="copy-compact-301", op="copy", layers=8, pages=640, pairs=301, kv_heads=16, page=64, head_dim=128,
             cache=E4M3, mix=10),
    ]


def log_int(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "beams", "beams", "copy"])
    if op == "beams":
        act = rng.choice([F32, F32, F16, BF16])
        vocab = log_int(rng, 1000, 152000)
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        most = max(1, int(MAX_LOGITS / (vocab * beams * (4 if act == F32 else 2))))
        return dict(op=op, requests=log_int(rng, 1, min(256, most)), beams=beams,
                    count=rng.choice([beams, beams, 2 * beams]), vocab=vocab, act=act, finished=rng.random() < 0.5)
    heads, kv_heads = rng.choice([(16, 16), (32, 8), (8, 1), (14, 2), (24, 8), (12, 12), (40, 8), (32, 32), (6, 2)])
    cache = rng.choice([INT8, E4M3])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128, 128]),
                page=rng.choice([16, 16, 32, 64, 128]), act=rng.choice([F16, BF16]), cache=cache,
                mix=rng.randrange(1 << 30))
    width = kv_heads * case["head_dim"]
    if op == "copy":
        layers = rng.choice([1, 2, 4, 8, 16])
        each = layers * width * case["page"] * 2  # bytes of one page's keys and values
        pairs = log_int(rng, 1, max(1, min(700, int(MAX_COPY / each))))
        return dict(op=op, layers=layers, pages=2 * pairs + rng.randint(1, 40), pairs=pairs, kv_heads=kv_heads,
                    page=case["page"], head_dim=case["head_dim"], cache=cache, mix=case["mix"])
    if op == "append":
        rows = log_int(rng, 1, 16384)
        requests = log_int(rng, 1, min(rows, 256))
        if cache == INT8:  # the cache is handed out as values: a small one
            requests = min(requests, 16)
            tokens = int(MAX_VALUES / width / requests)
            new = max(1, min(rows // requests, tokens // 2))
            kv = new + rng.randint(0, max(0, min(100, tokens - new - case["page"])))
        else:
            new = max(1, rows // requests)
            kv = new + log_int(rng, 1, 4096)
        case.update(requests=requests, new=new, kv=kv, norm=rng.random() < 0.5 and heads * case["head_dim"] <= 4096)
        return case
    kind = rng.choice(["decode", "verify", "mixed", "prefill"])
    requests = log_int(rng, 1, 128 if kind in ("decode", "verify") else 16)
    kv = log_int(rng, 16, max(16, min(65536, int(MAX_CACHE / (2 * width) / requests))))
    if kind == "decode":
        new = 1
    elif kind == "verify":
        new = rng.randint(2, 12)
    else:
        new = log_int(rng, 13, 4096)
        kv = min(kv, 16384)
    new = min(new, kv)
    if kind == "prefill":
        kv = new
    while requests > 1 and requests * new * kv * heads > MAX_SCORES:
        requests -= 1
    while requests * new * kv * heads > MAX_SCORES:
        new = max(1, new // 2)
        kv = new if kind == "prefill" else kv
    case.update(requests=requests, new=new, kv=kv, ragged=kind == "mixed" or rng.random() < 0.5)
    return case


def lengths(case):
    """(new tokens, tokens in all) of each request, from the case alone."""
    if not case.get("ragged"):
        # Appended tokens end at different places of their blocks.
        step = 1 if case["op"] == "append" and case["kv"] - case["new"] >= case["requests"] else 0
        return [(case["new"], case["kv"] - step * i) for i in range(case["requests"])]
    r = random.Random(case["mix"])
    got = []
    for _ in range(case["requests"]):
        kv = max(1, int(case["kv"] * math.exp(-r.random() * math.log(16))))
        new = case["new"]
        if new > 12:  # chunks beside requests that decode
            new = 1 if r.random() < 0.5 else r.randint(1, new)
        got.append((min(new, kv), kv))
    return got


def work(case):
    if case["op"] == "beams":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": n * (4 if case["act"] == F32 else 2) + case["requests"] * (5 * case["beams"] + 16 * case["count"]),
                "flops": 4 * n}
    D, token = case["head_dim"], case["kv_heads"] * 2 * (case["head_dim"] + 4 / BLOCK)
    if case["op"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["page"] * token, "flops": 0}
    lens = lengths(case)
    rows = sum(n for n, _ in lens)
    if case["op"] == "append":
        values = rows * (case["heads"] + 2 * case["kv_heads"]) * D
        return {"bytes": 2 * values + rows * (2 * case["heads"] * D + token + 8), "flops": 10 * values}
    pairs = sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in lens)
    seen = sum(kv for _, kv in lens)
    return {"bytes": 2 * rows * case["heads"] * D * 2 + seen * token, "flops": 4 * pairs * case["heads"] * D}


# ---------------------------------------------------------------------------
# inputs


def coded(x, cache):
    """[..., tokens, D] fp32 -> codes and the scales of its blocks of 16 tokens."""
    blocks = x.unflatten(-2, (-1, BLOCK))
    scales = blocks.abs().amax((-1, -2)) / LARGEST[cache]
    y = blocks.div_(scales[..., None, None])
    y = y.round_().to(torch.int8) if cache == INT8 else y.to(torch.float8_e4m3fn)
    return y.flatten(-3, -2), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
        return x.mul_(std) if std != 1.0 else x

    s = {"op": case["op"], "case": dict(case)}
    if case["op"] == "beams":
        R, beams = case["requests"], case["beams"]
        s["logits"] = normal(R, beams, case["vocab"], std=2.5).to(DTYPES[case["act"]])
        # Log probabilities of a few dozen tokens; beams of a request lie close together.
        s["scores"] = normal(R, 1, std=20.0) - 60 + normal(R, beams, std=1.5)
        s["finished"] = torch.rand(R, beams, generator=g, device="cuda") < 0.2 if case["finished"] else None
        return s
    Hk, D, page, cache = case["kv_heads"], case["head_dim"], case["page"], case["cache"]

    def pages_of(*shape):
        got = [coded(normal(*shape, Hk, page, D), cache) for _ in range(2)]
        (s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"]) = got

    if case["op"] == "copy":
        # Layer by layer: the fp32 values of a whole cache would take four times its room.
        for n in "kv":
            codes = torch.empty(case["layers"], case["pages"], Hk, page, D, dtype=DTYPES[cache], device="cuda")
            scales = torch.empty(case["layers"], case["pages"], Hk, page // BLOCK, device="cuda")
            for l in range(case["layers"]):
                codes[l], scales[l] = coded(normal(case["pages"], Hk, page, D), cache)
            s[n + "_pages"], s[n + "_scales"] = codes, scales
        order = list(range(case["pages"]))
        random.Random(seed ^ case["mix"]).shuffle(order)
        s["src"], s["dst"] = order[: case["pairs"]], order[case["pairs"]: 2 * case["pairs"]]
        return s
    lens = lengths(case)
    H = case["heads"]
    rows = sum(n for n, _ in lens)
    need = [-(-kv // page) for _, kv in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)[: sum(need)]
    starts = torch.tensor([0] + need).cumsum(0)[:-1]
    n_pages = torch.tensor(need)
    slot = torch.arange(max(need))
    inside = slot[None] < n_pages[:, None]
    at = (starts[:, None] + slot[None]).clamp(max=sum(need) - 1).cuda()
    s["page_table"] = torch.where(inside.cuda(), order[at], 0).to(torch.int32).contiguous()
    act = DTYPES[case["act"]]
    # Pages hold what was written before; a page's end past its request's
    # length holds a former owner's codes.
    pages_of(pages)
    new = torch.tensor([n for n, _ in lens])
    kv = torch.tensor([k for _, k in lens])
    s["requests"] = torch.repeat_interleave(torch.arange(len(lens)), new).to(torch.int32).cuda()
    first = new.cumsum(0) - new
    offset = torch.arange(rows) - torch.repeat_interleave(first, new)
    s["positions"] = (torch.repeat_interleave(kv - new, new) + offset).to(torch.int32).cuda()
    if case["op"] == "append":
        # A few tokens are larger than what their blocks hold, so that scales move.
        s["qkv"] = (normal(rows, (H + 2 * Hk) * D) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))).to(act)
        if case["norm"]:
            s["q_norm"] = 1 + normal(H * D, dtype=torch.float16, std=0.1)
            s["k_norm"] = 1 + normal(Hk * D, dtype=torch.float16, std=0.1)
        else:
            s["q_norm"] = s["k_norm"] = None
    else:
        # Scores with a standard deviation of two: neither flat nor one-hot.
        s["q"] = normal(rows, H, D, dtype=act, std=2.0)
        s["new"], s["kv"], s["first"] = new.cuda(), kv.cuda(), first.cuda()
        if own:  # the plan that a serving loop makes once a step and uses in every layer
            from trifuse_b200 import ops
            s["plan"] = ops.PagedPlan([n for n, _ in lens], [k for _, k in lens], H, Hk, D, page)
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    return run_own(s) if own else PLAIN[s["op"]](s)


def run_own(s):
    from trifuse_b200 import ops
    c = s["case"]
    if s["op"] == "beams":
        r = ops.beam_select(s["logits"], s["scores"], c["count"], finished=s["finished"], end=0)
        return {"score": r.score, "parent": r.parent, "token": r.token}
    caches = [s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]
    if s["op"] == "copy":
        ops.paged_copy(caches, s["src"], s["dst"])
        return held(s)
    if s["op"] == "append":
        q = ops.paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["page_table"], s["positions"], s["requests"],
                             c["heads"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rope_theta=THETA,
                             k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"q": q, **held(s)}
    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["plan"],
                               k_scales=s["k_scales"], v_scales=s["v_scales"])


def held(s):
    """The cache as outputs: 8-bit floating codes with their scales; whole-number
    codes that were computed as the values that they stand for; whole-number codes
    that were copied as they are."""
    got = {n: s[n] for n in ("k_scales", "v_scales")}
    if s["op"] == "append" and s["case"]["cache"] == INT8:
        for n in "kv":
            got[n] = values(s[n + "_pages"], s[n + "_scales"]).to(DTYPES[s["case"]["act"]])
    else:
        got.update(k_pages=s["k_pages"], v_pages=s["v_pages"])
    return got


def values(codes, scales):
    """fp32 values of codes [..., tokens, D] with scales [..., blocks]."""
    return (codes.float().unflatten(-2, (-1, BLOCK)) * scales[..., None, None]).flatten(-3, -2)


def plain_norm_rope(x, weight, positions, heads, D):
    """x [rows, heads * D] fp32 -> normalised over the full width, rotated by halves."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    x = x.view(x.shape[0], heads, D)
    inv = THETA ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=torch.float64) / D)
    angle = positions.double()[:, None] * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., : D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def plain_append(s):
    c = s["case"]
    H, Hk, D, page, cache = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["cache"]
    q, k, v = s["qkv"].float().split([H * D, Hk * D, Hk * D], -1)
    q = plain_norm_rope(q, s["q_norm"], s["positions"], H, D)
    k = plain_norm_rope(k, s["k_norm"], s["positions"], Hk, D)
    at, pos = s["requests"].long(), s["positions"].long()
    # The blocks that new tokens fall into, each row's block, and the blocks' first new slots.
    name, block = torch.unique_consecutive(at * (1 << 32) + pos // BLOCK, return_inverse=True)
    n = name.shape[0]
    first = torch.full((n,), BLOCK, device="cuda").scatter_reduce(0, block, pos % BLOCK, "amin")
    number = name % (1 << 32)
    where = s["page_table"][name >> 32, number * BLOCK // page].long()
    part = number % (page // BLOCK)
    for pages, scales, x in ((s["k_pages"], s["k_scales"], k), (s["v_pages"], s["v_scales"], v.reshape(-1, Hk, D))):
        old = torch.where((first > 0)[:, None], scales[where, :, part], 0.0)
        most = torch.zeros(n, Hk, device="cuda").scatter_reduce(0, block[:, None].expand(-1, Hk), x.abs().amax(-1),
                                                                "amax")
        scale = torch.maximum(old, most / LARGEST[cache])
        # [blocks, heads, slots, D]: what is there, at the new scale, with the new tokens put in.
        split = pages.view(-1, Hk, page // BLOCK, BLOCK, D)
        y = split[where, :, part].float()
        earlier = torch.arange(BLOCK, device="cuda") < first[:, None]
        moved = y * (old / scale)[..., None, None]
        y = torch.where(earlier[:, None, :, None], moved, y)
        y[block, :, pos % BLOCK] = x / scale[block][..., None]
        y = y.round().to(torch.int8) if cache == INT8 else y.to(torch.float8_e4m3fn)
        split[where, :, part] = y
        scales[where, :, part] = scale
    return {"q": q.to(s["qkv"].dtype), **held(s)}


def plain_attention(s):
    c = s["case"]
    H, Hk, D = c["heads"], c["kv_heads"], c["head_dim"]
    lens = lengths(c)
    B, G, N = len(lens), H // Hk, max(n for n, _ in lens)
    rows = s["q"].shape[0]
    # queries padded to [B, kv head, token, group head, D]
    at = (s["first"][:, None] + torch.arange(N, device="cuda")).clamp(max=rows - 1)
    q = s["q"].float()[at].view(B, N, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, N * G, D)

    def history(pages, scales):  # [B, kv head, token, D]
        ids = s["page_table"].long()
        x = values(pages[ids], scales[ids])  # [B, pages, kv head, slot, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)

    score = (q @ history(s["k_pages"], s["k_scales"]).transpose(-1, -2)).mul_(D ** -0.5).view(B, Hk, N, G, -1)
    key = torch.arange(score.shape[-1], device="cuda")
    last = s["kv"][:, None] - s["new"][:, None] + torch.arange(N, device="cuda")  # last key of each query
    hidden = key[None, None] > last[..., None]  # [B, N, keys]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(B, Hk, N * G, -1) @ history(s["v_pages"], s["v_scales"])).view(B, Hk, N, G, D) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(B, N, H, D)
    return out[s["requests"].long(), s["positions"].long() - (s["kv"] - s["new"])[s["requests"].long()]].to(
        s["q"].dtype)


def plain_beams(s):
    # In 64 bits: which of two near continuations comes first must not hang on a rounding.
    x, count = s["logits"].double(), s["case"]["count"]
    R, beams, V = x.shape
    m = x.amax(-1, keepdim=True)
    total = s["scores"].double()[..., None] + (x - m - (x - m).exp().sum(-1, keepdim=True).log())
    if s["finished"] is not None:  # an ended beam goes on as it is, with the end token
        ended = torch.full_like(total, -math.inf)
        ended[..., 0] = s["scores"].double()
        total = torch.where(s["finished"][..., None], ended, total)
    best, index = torch.sort(total.view(R, beams * V), dim=-1, descending=True, stable=True)
    best, index = best[:, :count].float(), index[:, :count]
    none = best == -math.inf  # fewer continuations than asked for
    return {"score": best, "parent": torch.where(none, -1, index // V).to(torch.int32),
            "token": torch.where(none, -1, index % V)}


def plain_copy(s):
    src, dst = (torch.tensor(s[n], device="cuda") for n in ("src", "dst"))
    for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
        x = s[n].view(torch.uint8) if s[n].element_size() == 1 else s[n]
        x[:, dst] = x[:, src]
    return held(s)


PLAIN = {"append": plain_append, "attention": plain_attention, "beams": plain_beams, "copy": plain_copy}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "beams":
        x, R = s["logits"].double(), case["requests"]
        p = torch.log_softmax(x, -1) + s["scores"].double()[..., None]
        if case["finished"]:
            f = s["finished"]
            p[f] = -math.inf
            p[..., 0][f] = s["scores"].double()[f]
        return {"score": p.reshape(R, -1).topk(case["count"], -1).values, "parent": None, "token": None}
    if case["op"] == "copy":
        for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
            for a, b in zip(s["src"], s["dst"]):
                s[n][:, b].copy_(s[n][:, a])
        return {n: s[n].double() if s[n].dtype != torch.int8 else None for n in
                ("k_pages", "v_pages", "k_scales", "v_scales")}
    lens = lengths(case)
    H, Hk, D, page, cache = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["cache"]
    table = s["page_table"].tolist()
    if case["op"] == "append":
        x = s["qkv"].double()
        turn = s["positions"].double()[:, None] / THETA ** (torch.arange(0, D, 2).double().cuda() / D)
        z = torch.polar(torch.ones_like(turn), turn)[:, None]

        def part(a, heads, w):
            if w is not None:
                a = a / (a.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            a = a.reshape(len(a), heads, 2, D // 2)
            r = torch.complex(a[:, :, 0], a[:, :, 1]) * z
            return torch.stack([r.real, r.imag], 2).reshape(len(a), heads, D)

        def code(a):
            return a.round() if cache == INT8 else a.float().to(torch.float8_e4m3fn).double()

        q = part(x[:, : H * D], H, s["q_norm"])
        k = part(x[:, H * D: (H + Hk) * D], Hk, s["k_norm"])
        v = x[:, (H + Hk) * D:].reshape(-1, Hk, D)
        got = {"q": q}
        for n, new in (("k", k), ("v", v)):
            codes, scales = s[n + "_pages"].double(), s[n + "_scales"].double()
            row = 0
            for b, (count, kv) in enumerate(lens):
                p = kv - count
                while p < kv:  # a block at a time
                    end = min(kv, p // BLOCK * BLOCK + BLOCK)
                    at, i, o = table[b][p // page], p % page // BLOCK, p % page
                    fresh = new[row: row + end - p].transpose(0, 1)  # [Hk, tokens, D]
                    scale = fresh.abs().amax((1, 2)) / LARGEST[cache]
                    if p % BLOCK:
                        before = scales[at, :, i].clone()
                        scale = torch.maximum(scale, before)
                        held_codes = codes[at, :, i * BLOCK: o]
                        codes[at, :, i * BLOCK: o] = code(held_codes * (before / scale)[:, None, None])
                    codes[at, :, o: o + end - p] = code(fresh / scale[:, None, None])
                    scales[at, :, i] = scale
                    row += end - p
                    p = end
            got[n + "_scales"] = scales
            if cache == INT8:
                got[n] = codes * scales.repeat_interleave(BLOCK, -1)[..., None]
            else:
                got[n + "_pages"] = codes
        return got
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    G, row = H // Hk, 0
    for b, (n, kv) in enumerate(lens):
        ids = torch.tensor(table[b][: -(-kv // page)], device="cuda")
        unseen = torch.ones(n, kv, dtype=torch.bool, device="cuda").triu(kv - n + 1)
        for h in range(Hk):
            k, v = ((s[x + "_pages"][ids, h].double() *
                     s[x + "_scales"][ids, h].double().repeat_interleave(BLOCK, -1)[..., None]).reshape(-1, D)[:kv]
                    for x in "kv")
            q = s["q"][row: row + n, h * G: (h + 1) * G].double()
            a = torch.einsum("ngd,kd->gnk", q, k) / math.sqrt(D)
            a = torch.softmax(a.masked_fill(unseen, -math.inf), -1)
            out[row: row + n, h * G: (h + 1) * G] = (a @ v).transpose(0, 1)
        row += n
    return out
