"""Measured cases of the paged serving operators: append, attention, token log probabilities.

The three run in this order in a serving step over a paged key/value cache.
``paged_append`` normalises and rotates the new tokens' queries and keys and
writes keys and values into the requests' pages.  ``paged_attention`` lets the
new tokens of every request attend that request's pages.  ``token_logprobs``
turns the step's logits into what an answer reports: the log probability of
given tokens, the entropy, the rank and the top alternatives.

``own`` selects between the plain torch form of each operator (False) and the
framework's kernels (True).
"""
import math
import random

import torch

own = False

F16, BF16, F32 = "f16", "bf16", "f32"
DTYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
EPS = 1e-5
THETA = 10000.0
# Cost bounds of a drawn case: what the largest listed cases reach.
MAX_SCORES = 2.3e9   # padded (head, query, key) triples of the plain form
MAX_CACHE = 2.2e9    # bytes of keys and values that one call sees
MAX_LOGITS = 4.2e8   # bytes of logits


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # One decode step of a batch of 64 requests: one new token each, full-width
        # query/key norms and rotation, float16 cache (this model's layer).
        dict(name="append-decode-64", op="append", requests=64, new=1, kv=4096, heads=16, kv_heads=16, head_dim=128,
             page=64, act=BF16, cache=F16, norm=True, mix=1),
        # A prefill of 8 prompts of 2048 tokens, the same layer.
        dict(name="append-prefill-16384", op="append", requests=8, new=2048, kv=2048, heads=16, kv_heads=16,
             head_dim=128, page=64, act=BF16, cache=F16, norm=True, mix=2),
        # One request's decode step on a short history: nothing but latency.
        dict(name="decode-1x600", op="attention", requests=1, new=1, kv=600, ragged=False, heads=16, kv_heads=16,
             head_dim=128, page=16, act=F16, cache=F16, mix=3),
        # The decode batch of this repository's benchmark: 64 requests at 4096 tokens.
        dict(name="decode-64x4096", op="attention", requests=64, new=1, kv=4096, ragged=False, heads=16, kv_heads=16,
             head_dim=128, page=64, act=BF16, cache=F16, mix=4),
        # A serving batch whose histories differ by a factor of sixteen, grouped heads.
        dict(name="decode-ragged-37", op="attention", requests=37, new=1, kv=32768, ragged=True, heads=32, kv_heads=8,
             head_dim=128, page=16, act=BF16, cache=BF16, mix=5),
        # Checking a few drafted tokens for each request: 5 new tokens, 7 query heads
        # on each key head, odd lengths, narrow heads.
        dict(name="verify-24x5", op="attention", requests=24, new=5, kv=8011, ragged=False, heads=14, kv_heads=2,
             head_dim=64, page=32, act=BF16, cache=BF16, mix=6),
        # Prompt chunks and decoding requests mixed in one step.
        dict(name="mixed-12", op="attention", requests=12, new=601, kv=8003, ragged=True, heads=32, kv_heads=8,
             head_dim=128, page=16, act=BF16, cache=BF16, mix=7),
        # The prefill of this repository's benchmark: 8 whole prompts of 2048 tokens.
        dict(name="prefill-8x2048", op="attention", requests=8, new=2048, kv=2048, ragged=False, heads=16, kv_heads=16,
             head_dim=128, page=64, act=F16, cache=F16, mix=8),
        # A late chunk of a long document: 2048 new tokens after 32768.
        dict(name="chunk-2048-of-34816", op="attention", requests=1, new=2048, kv=34816, ragged=False, heads=32,
             kv_heads=8, head_dim=128, page=128, act=BF16, cache=BF16, mix=9),
        # One generated token of one request, with twenty alternatives.
        dict(name="logprobs-1", op="logprobs", rows=1, vocab=50304, top=20, act=F32),
        # One step of a decode batch.
        dict(name="logprobs-64", op="logprobs", rows=64, vocab=50304, top=20, act=F32),
        # Scoring the tokens of long prompts (one row short of a round number).
        dict(name="logprobs-4095", op="logprobs", rows=4095, vocab=50304, top=5, act=BF16),
    ]


def log_int(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "logprobs"])
    if op == "logprobs":
        act = rng.choice([F32, F32, F16, BF16])
        vocab = log_int(rng, 1000, 152000)
        most = max(1, int(MAX_LOGITS / (vocab * (4 if act == F32 else 2))))
        return dict(op=op, rows=log_int(rng, 1, min(4096, most)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 64]),
                    act=act)
    heads, kv_heads = rng.choice([(16, 16), (32, 8), (8, 1), (14, 2), (24, 8), (12, 12), (40, 8), (32, 32), (6, 2)])
    act, cache = rng.choice([(F16, F16), (BF16, BF16), (BF16, F16)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128, 128]),
                page=rng.choice([16, 16, 32, 64, 128]), act=act, cache=cache, mix=rng.randrange(1 << 30))
    if op == "append":
        rows = log_int(rng, 1, 16384)
        requests = log_int(rng, 1, min(rows, 256))
        new = max(1, rows // requests)
        case.update(requests=requests, new=new, kv=new + log_int(rng, 1, 4096),
                    norm=rng.random() < 0.5 and heads * case["head_dim"] <= 4096)
        return case
    kind = rng.choice(["decode", "verify", "mixed", "prefill"])
    token = 4 * kv_heads * case["head_dim"]  # bytes of one token's key and value
    requests = log_int(rng, 1, 128 if kind in ("decode", "verify") else 16)
    kv = log_int(rng, 16, max(16, min(65536, int(MAX_CACHE / token / requests))))
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
        return [(case["new"], case["kv"])] * case["requests"]
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
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["act"] == F32 else 2) + case["rows"] * (20 + 12 * case["top"]), "flops": 6 * n}
    lens = lengths(case)
    rows, D = sum(n for n, _ in lens), case["head_dim"]
    if case["op"] == "append":
        values = rows * (case["heads"] + 2 * case["kv_heads"]) * D
        return {"bytes": 2 * values * 2 + 8 * rows, "flops": 8 * values}
    pairs = sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in lens)
    seen = sum(kv for _, kv in lens)
    return {"bytes": 2 * rows * case["heads"] * D * 2 + 2 * seen * case["kv_heads"] * D * 2,
            "flops": 4 * pairs * case["heads"] * D}


# ---------------------------------------------------------------------------
# inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype, std=1.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
        return x.mul_(std) if std != 1.0 else x

    s = {"op": case["op"], "case": dict(case)}
    if case["op"] == "logprobs":
        # Logits with a spread like a trained model's; the given tokens are drawn
        # from the distribution that the logits stand for.
        x = normal(case["rows"], case["vocab"], dtype=torch.float32, std=2.5)
        u = torch.rand(x.shape, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
        s["tokens"] = (x - (-u.log()).log()).argmax(-1)
        s["logits"] = x.to(DTYPES[case["act"]])
        return s
    lens = lengths(case)
    H, Hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
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
    act, cache = DTYPES[case["act"]], DTYPES[case["cache"]]
    # Pages hold what was written before; a page's end past its request's
    # length holds a former owner's values.
    s["k_pages"] = normal(pages, Hk, page, D, dtype=cache)
    s["v_pages"] = normal(pages, Hk, page, D, dtype=cache)
    new = torch.tensor([n for n, _ in lens])
    kv = torch.tensor([k for _, k in lens])
    s["requests"] = torch.repeat_interleave(torch.arange(len(lens)), new).to(torch.int32).cuda()
    first = new.cumsum(0) - new
    offset = torch.arange(rows) - torch.repeat_interleave(first, new)
    s["positions"] = (torch.repeat_interleave(kv - new, new) + offset).to(torch.int32).cuda()
    if case["op"] == "append":
        s["qkv"] = normal(rows, (H + 2 * Hk) * D, dtype=act)
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
    if s["op"] == "append":
        q = ops.paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["page_table"], s["positions"], s["requests"],
                             s["case"]["heads"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rope_theta=THETA)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["op"] == "attention":
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["plan"])
    r = ops.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank, "top_logprob": r.top_logprob,
            "top_token": r.top_token}


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
    H, Hk, D, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    q, k, v = s["qkv"].float().split([H * D, Hk * D, Hk * D], -1)
    q = plain_norm_rope(q, s["q_norm"], s["positions"], H, D)
    k = plain_norm_rope(k, s["k_norm"], s["positions"], Hk, D)
    at, pos = s["requests"].long(), s["positions"].long()
    where = s["page_table"][at, pos // page].long()
    s["k_pages"][where, :, pos % page] = k.to(s["k_pages"].dtype)
    s["v_pages"][where, :, pos % page] = v.view(-1, Hk, D).to(s["v_pages"].dtype)
    return {"q": q.to(s["qkv"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def plain_attention(s):
    c = s["case"]
    H, Hk, D = c["heads"], c["kv_heads"], c["head_dim"]
    lens = lengths(c)
    B, G, N = len(lens), H // Hk, max(n for n, _ in lens)
    rows = s["q"].shape[0]
    # queries padded to [B, kv head, token, group head, D]
    at = (s["first"][:, None] + torch.arange(N, device="cuda")).clamp(max=rows - 1)
    q = s["q"].float()[at].view(B, N, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, N * G, D)

    def history(pages):  # [B, kv head, token, D]
        x = pages[s["page_table"].long()]  # [B, pages, kv head, slot, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D).float()

    score = (q @ history(s["k_pages"]).transpose(-1, -2)).mul_(D ** -0.5).view(B, Hk, N, G, -1)
    key = torch.arange(score.shape[-1], device="cuda")
    last = s["kv"][:, None] - s["new"][:, None] + torch.arange(N, device="cuda")  # last key of each query
    hidden = key[None, None] > last[..., None]  # [B, N, keys]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(B, Hk, N * G, -1) @ history(s["v_pages"])).view(B, Hk, N, G, D) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(B, N, H, D)
    return out[s["requests"].long(), s["positions"].long() - (s["kv"] - s["new"])[s["requests"].long()]].to(
        s["q"].dtype)


def plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    given = x.gather(-1, s["tokens"][:, None])
    index = torch.arange(x.shape[1], device="cuda")
    before = (x > given) | ((x == given) & (index[None] < s["tokens"][:, None]))
    best, token = torch.sort(x, dim=-1, descending=True, stable=True)  # ties to the lowest index
    return {"logprob": (given - lse)[:, 0], "entropy": (lse - (e * x).sum(-1, keepdim=True) / total)[:, 0],
            "rank": before.sum(-1).to(torch.int32), "top_logprob": (best[:, :top] - lse).contiguous(),
            "top_token": token[:, :top].contiguous()}


PLAIN = {"append": plain_append, "attention": plain_attention, "logprobs": plain_logprobs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1)
        p = torch.softmax(x, -1)
        entropy = -torch.xlogy(p, p).sum(-1)
        t = torch.topk(x, case["top"], -1).values - lse[:, None]
        return {"logprob": x[torch.arange(x.shape[0]), s["tokens"]] - lse, "entropy": entropy, "rank": None,
                "top_logprob": t, "top_token": None}
    lens = lengths(case)
    H, Hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
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

        q = part(x[:, : H * D], H, s["q_norm"])
        k = part(x[:, H * D: (H + Hk) * D], Hk, s["k_norm"])
        v = x[:, (H + Hk) * D:].reshape(-1, Hk, D)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        slots, row = [], 0
        for b, (n, kv) in enumerate(lens):
            slots += [table[b][p // page] * page + p % page for p in range(kv - n, kv)]
        slots = torch.tensor(slots, device="cuda")
        for pages, new in ((k_pages, k), (v_pages, v)):
            flat = pages.transpose(1, 2).reshape(-1, Hk, D)
            flat[slots] = new
            pages.copy_(flat.view(-1, page, Hk, D).transpose(1, 2))
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    G, row = H // Hk, 0
    for b, (n, kv) in enumerate(lens):
        ids = torch.tensor(table[b][: -(-kv // page)], device="cuda")
        unseen = torch.ones(n, kv, dtype=torch.bool, device="cuda").triu(kv - n + 1)
        for h in range(Hk):
            k = s["k_pages"][ids, h].reshape(-1, D)[:kv].double()
            v = s["v_pages"][ids, h].reshape(-1, D)[:kv].double()
            q = s["q"][row: row + n, h * G: (h + 1) * G].double()
            a = torch.einsum("ngd,kd->gnk", q, k) / math.sqrt(D)
            a = torch.softmax(a.masked_fill(unseen, -math.inf), -1)
            out[row: row + n, h * G: (h + 1) * G] = (a @ v).transpose(0, 1)
        row += n
    return out
