"""Paged append and paged attention against their formulas in 64 bits.

Tolerances are derived from the roundings on the way.  Append computes in
fp32 and rounds once, so a value may be off by half a unit of its 16-bit type
plus a few fp32 roundings.  Attention rounds each weight p (relative 2^-11 in
f16, 2^-8 in bf16) and the output once; the weights' roundings add up to at
most u * sum p |v| / sum p <= u * max |v| of the visible values, so an output
is within u * max |v| + u * |out| plus fp32 noise (the scores' products of
16-bit values are summed in fp32: 1e-4 relative covers them and the cubic
exponential where one is used)."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def make_cache(lens, kv_heads, D, page, dtype, seed=0, spare=3, fill=None):
    """Shuffled pages for the lengths: (k_pages, v_pages, page table); slots past a length hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    k = torch.randn(pages, kv_heads, page, D, generator=g).to(dtype)
    v = torch.randn(pages, kv_heads, page, D, generator=g).to(dtype)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n].to(torch.int32)
        at += n
        if fill is not None and lens[r] % page:
            k[order[at - 1], :, lens[r] % page:] = fill
            v[order[at - 1], :, lens[r] % page:] = fill
    return k.cuda(), v.cuda(), table.cuda()


def history(pages, table, r, n, page):
    """[n, kv_heads, D] in float64."""
    ids = table[r, : -(-n // page)].long()
    x = pages[ids].double().transpose(1, 2)
    return x.reshape(-1, *x.shape[2:])[:n]


def reference(q, k_pages, v_pages, table, new, kv, scale=None):
    H, D = q.shape[1:]
    Hk, page = k_pages.shape[1:3]
    G = H // Hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    big = torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
    row = 0
    for r, (n, L) in enumerate(zip(new, kv)):
        if n and L:
            k, v = history(k_pages, table, r, L, page), history(v_pages, table, r, L, page)
            qq = q[row:row + n].double().view(n, Hk, G, D)
            s = torch.einsum("nhgd,khd->nhgk", qq, k) * (D ** -0.5 if scale is None else scale)
            hidden = torch.arange(L, device=q.device)[None] > (L - n + torch.arange(n, device=q.device))[:, None]
            s = s.masked_fill(hidden[:, None, None], -np.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.where(s == -np.inf, 0.0, torch.exp(s - torch.where(m == -np.inf, 0.0, m)))
            l = e.sum(-1, keepdim=True)
            o = torch.einsum("nhgk,khd->nhgd", e / torch.where(l == 0, 1.0, l), v)
            out[row:row + n] = o.reshape(n, H, D)
            big[row:row + n] = v.abs().max()
        row += n
    return out, big


def check(got, want, big, cache):
    assert got.dtype in UNIT
    err = (got.double() - want).abs()
    bound = UNIT[cache] * big[:, None, None] + UNIT[got.dtype] * want.abs() + 1e-4 * big[:, None, None] + 1e-6
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.2f} of the bound"


def run(ops, new, kv, H, Hk, D, page, act, cache, seed=0, fill=float("nan"), scale=None):
    k, v, table = make_cache(kv, Hk, D, page, cache, seed, fill=fill)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(sum(new), H, D, generator=g) * 2).to(act).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    got = ops.paged_attention(q, k, v, table, plan, scale=scale)
    assert ops.device_error() == 0
    want, big = reference(q, k, v, table, new, kv, scale)
    check(got, want, big, cache)
    return q, k, v, table, plan, got


TYPES = [(F16, F16), (BF16, BF16), (BF16, F16)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(16, 16), (8, 1), (14, 2), (6, 2)])
def test_decode(ops, act, cache, D, H, Hk):
    """Single tokens, from one key to several splits, lengths around tile and page ends."""
    run(ops, [1] * 9, [1, 2, 15, 16, 17, 32, 33, 600, 5003], H, Hk, D, 16, act, cache)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_page_sizes(ops, page):
    run(ops, [1, 3, 1, 2], [7, 300, 257, 1025], 8, 2, 128, page, BF16, BF16)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("D,H,Hk", [(128, 16, 16), (64, 14, 2), (128, 32, 8), (128, 5, 1), (64, 6, 6)])
def test_chunks(ops, act, cache, D, H, Hk):
    """Chunks of many lengths in one call: whole prompts, late chunks, single tokens, an idle request."""
    run(ops, [1, 130, 0, 257, 1, 77, 300], [900, 130, 50, 1300, 1, 500, 2049], H, Hk, D, 16, act, cache)


@pytest.mark.parametrize("n", [1, 2, 3, 16, 17, 33, 64, 127, 128, 129, 255, 256, 257, 511])
def test_prompt_lengths(ops, n):
    run(ops, [n], [n], 4, 2, 128, 32, F16, F16, seed=n)


@pytest.mark.parametrize("n,L", [(1, 127), (1, 128), (1, 129), (5, 4096), (40, 4097), (128, 8191), (300, 20000)])
def test_long_history(ops, n, L):
    """Few rows over a long history: the keys are divided and the parts merged."""
    run(ops, [n], [L], 8, 2, 128, 64, BF16, BF16, seed=L)


def test_rows_that_attend_nothing(ops):
    """kv shorter than the new tokens: the rows before token 0 give zeros; so does an empty history."""
    for new, kv in (([5], [3]), ([1, 4], [0, 0]), ([40, 300], [30, 0]), ([200], [70])):
        *_, got = run(ops, new, kv, 8, 2, 128, 16, F16, F16)
        n, L = new[0], kv[0]
        assert (got[: max(0, n - L)] == 0).all()


def test_plan_takes_other_integers(ops):
    """Lengths as tensors and numpy arrays; a length that would wrap is refused."""
    import numpy as np
    a = ops.PagedPlan(torch.tensor([1, 5]), np.array([40, 60]), 4, 2, 64, 16)
    assert a.positions.tolist() == [39, 55, 56, 57, 58, 59]
    with pytest.raises(ValueError):
        ops.PagedPlan([1], [(1 << 32) + 5], 4, 2, 64, 16)
    with pytest.raises(ValueError):
        ops.PagedPlan([1, 2], [5], 4, 2, 64, 16)


def test_no_rows(ops):
    k, v, table = make_cache([10, 0], 2, 64, 16, F16)
    plan = ops.PagedPlan([0, 0], [10, 0], 4, 2, 64, 16)
    assert ops.paged_attention(torch.empty(0, 4, 64, dtype=F16, device="cuda"), k, v, table, plan).shape == (0, 4, 64)
    plan = ops.PagedPlan([], [], 4, 2, 64, 16)
    assert plan.rows == 0


@pytest.mark.parametrize("n", [1, 40, 300])
def test_nan_and_infinite_scores(ops, n):
    """A NaN or +inf score makes its rows NaN, a -inf score drops its key; other rows keep their values."""
    L, H, Hk, D = 700, 4, 2, 128
    for bad in (float("nan"), float("inf"), -float("inf")):
        k, v, table = make_cache([L], Hk, D, 16, F16)
        q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
        q[..., 0] = 1.0
        at = [3, L - 1 - n // 2] if n > 1 else [3, 300]
        for t in at[1:]:
            k[table[0, t // 16].long(), 0, t % 16, 0] = bad
        plan = ops.PagedPlan([n], [L], H, Hk, D, 16)
        got = ops.paged_attention(q, k, v, table, plan)
        want, big = reference(q, k, v, table, [n], [L])
        seen = torch.arange(n, device="cuda") + L - n >= at[1]
        if bad == -float("inf"):
            check(got, want, big, F16)
        else:
            assert torch.isnan(got[seen][:, : H // Hk]).all()
            clean = got.clone()
            clean[seen, : H // Hk] = 0
            want[seen, : H // Hk] = 0
            check(clean, want, big, F16)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,Hk,D,n,L", [(4, 4, 64, 2, 2), (4, 4, 128, 16, 700), (6, 2, 128, 5, 333), (8, 2, 64, 4, 5000),
                                        (4, 2, 128, 40, 700), (2, 2, 64, 128, 9000), (4, 4, 128, 300, 300),
                                        (4, 1, 128, 150, 6000), (3, 3, 64, 513, 900)])
def test_masked_values_that_are_not_finite(ops, act, cache, H, Hk, D, n, L):
    """A NaN or infinite value reaches the rows that see its token, in its column of its key head, and
    nothing else changes by a bit."""
    G, page = H // Hk, 16
    k, v, table = make_cache([L, L], Hk, D, page, cache)
    q = torch.randn(2 * n, H, D, generator=torch.Generator().manual_seed(3)).to(act).cuda()
    plan = ops.PagedPlan([n, n], [L, L], H, Hk, D, page)
    spots = [(0, L - 1, float("nan"), 0, 1), (0, L - 1 - n // 3, float("inf"), Hk - 1, D - 1),
             (1, L - 1 - n // 2, -float("inf"), 0, D // 2 + 3), (1, L - n, float("nan"), Hk - 1, 7)]
    for r, t, _, h, d in spots:
        v[table[r, t // page].long(), h, t % page, d] = 0
    clean = ops.paged_attention(q, k, v, table, plan)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for r, t, bad, h, d in spots:
        v[table[r, t // page].long(), h, t % page, d] = bad
        first = n * r + t - (L - n)
        hit[first:n * (r + 1), h * G:(h + 1) * G, d] = True
    got = ops.paged_attention(q, k, v, table, plan)
    assert ops.device_error() == 0
    assert torch.isfinite(clean).all() and not torch.isfinite(got[hit]).any()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("n", [1, 200])
def test_every_score_minus_infinity(ops, n):
    k, v, table = make_cache([n], 2, 64, 16, BF16)
    k.zero_()
    k[..., 0] = -float("inf")
    q = torch.ones(n, 4, 64, dtype=BF16, device="cuda")
    plan = ops.PagedPlan([n], [n], 4, 2, 64, 16)
    assert (ops.paged_attention(q, k, v, table, plan) == 0).all()


@pytest.mark.parametrize("n", [1, 150])
def test_large_scores(ops, n):
    """Scores far apart: the maximum moves late and by much, and small weights vanish."""
    L, D = 1000, 128
    k, v, table = make_cache([L], 2, D, 16, F16)
    ramp = torch.linspace(-60, 60, L)
    for t in range(L):
        k[table[0, t // 16].long(), :, t % 16] = ramp[t].to(F16)
    q = torch.full((n, 4, D), 0.25, dtype=F16, device="cuda")
    plan = ops.PagedPlan([n], [L], 4, 2, D, 16)
    got = ops.paged_attention(q, k, v, table, plan)
    want, big = reference(q, k, v, table, [n], [L])
    check(got, want, big, F16)


@pytest.mark.parametrize("n", [1, 60])
def test_strides_and_interleaved_pages(ops, n):
    """q as a slice of a fused projection, k and v pages in one buffer, a page table that is a view."""
    H, Hk, D, page, L = 8, 2, 128, 16, 333
    k, v, table = make_cache([L, L], Hk, D, page, F16)
    both = torch.full((k.shape[0], 2, Hk, page, D), float("nan"), dtype=F16, device="cuda")
    both[:, 0], both[:, 1] = k, v
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    fused = torch.randn(2 * n, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(5)).to(F16).cuda()
    q = fused[:, : H * D].view(2 * n, H, D)
    plan = ops.PagedPlan([n, n], [L, L], H, Hk, D, page)
    want = ops.paged_attention(q.contiguous(), k, v, table, plan)
    got = ops.paged_attention(q, both[:, 0], both[:, 1], wide[:, 2:2 + table.shape[1]], plan)
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    assert ops.paged_attention(q, k, v, table, plan, out=out) is out and torch.equal(out, want)


def test_rows_off_their_alignment(ops):
    """q and qkv views that start in the middle of a 16-byte vector, or whose rows do."""
    H, Hk, D, page, L = 4, 2, 64, 16, 40
    k, v, table = make_cache([L], Hk, D, page, F16)
    plan = ops.PagedPlan([3], [L], H, Hk, D, page)
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(3, (H + 2 * Hk) * D + 13, generator=g).to(F16).cuda()
    qkv = wide[:, 3:3 + (H + 2 * Hk) * D]
    k2, v2 = k.clone(), v.clone()
    q = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H)
    assert torch.equal(q, ops.paged_append(qkv.contiguous(), k2, v2, table, plan.positions, plan.requests, H))
    assert torch.equal(k, k2) and torch.equal(v, v2)
    view = wide[:, 3:3 + H * D].view(3, H, D)
    assert torch.equal(ops.paged_attention(view, k, v, table, plan),
                       ops.paged_attention(view.contiguous(), k, v, table, plan))


def test_repeatable_and_plan_reused(ops):
    """The same plan again gives the same bits (parts merge in a fixed order, counters are left zero)."""
    q, k, v, table, plan, got = run(ops, [1, 30, 300, 1], [9000, 4000, 5000, 17], 8, 2, 128, 16, BF16, BF16)
    for _ in range(20):
        assert torch.equal(ops.paged_attention(q, k, v, table, plan), got)


def test_other_stream(ops):
    new, kv = [1, 50], [3000, 700]
    k, v, table = make_cache(kv, 2, 128, 16, F16)
    q = torch.randn(51, 8, 128, generator=torch.Generator().manual_seed(2)).to(F16).cuda()
    plan = ops.PagedPlan(new, kv, 8, 2, 128, 16)
    want = ops.paged_attention(q, k, v, table, plan)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        plan2 = ops.PagedPlan(new, kv, 8, 2, 128, 16)
        a = ops.paged_attention(q, k, v, table, plan2)
    b = ops.paged_attention(q, k, v, table, plan2)  # made on s, used here
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_graph_capture(ops):
    new, kv = [1, 1, 90], [3000, 33, 700]
    k, v, table = make_cache(kv, 2, 128, 16, F16)
    q = torch.randn(92, 8, 128, generator=torch.Generator().manual_seed(2)).to(F16).cuda()
    plan = ops.PagedPlan(new, kv, 8, 2, 128, 16)
    want = ops.paged_attention(q, k, v, table, plan)
    out = torch.zeros_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ops.paged_attention(q, k, v, table, plan, out=out)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_pages_beyond_a_gigabyte(ops):
    """Byte offsets past 32 bits: a cache of over 4 GB whose used pages are the last ones."""
    pages, Hk, page, D = 9000, 16, 128, 128  # 4.7 GB a side
    k = torch.zeros(pages, Hk, page, D, dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    L = 700
    table = torch.arange(pages - 6, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    qkv = torch.randn(L, 3 * Hk * D, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    for new in ([L], [1]):
        plan = ops.PagedPlan(new, [L], Hk, Hk, D, page)
        n = new[0]
        q = ops.paged_append(qkv[:n], k, v, table, plan.positions, plan.requests, Hk)
        got = ops.paged_attention(q, k, v, table, plan)
        want, big = reference(q, k, v, table, new, [L])
        check(got, want, big, F16)
    assert (k[0] == 0).all()


# ---------------------------------------------------------------- append


def append_reference(qkv, H, Hk, D, positions, qn, kn, eps, theta):
    x = qkv.double()
    q, k, v = x[:, : H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:]

    def turn(a, heads, w):
        if w is not None:
            a = a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps) * w.double()
        a = a.reshape(len(a), heads, D)
        if theta is None:
            return a
        t = positions.double()[:, None] * theta ** (-torch.arange(0, D, 2, device=a.device).double() / D)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        lo, hi = a[..., : D // 2], a[..., D // 2:]
        return torch.cat([lo * c - hi * s, lo * s + hi * c], -1)

    return turn(q, H, qn), turn(k, Hk, kn), v.reshape(len(v), Hk, D)


def near(got, want):
    """Half a unit of the 16-bit type (2^-11 / 2^-8 of the value, or of the smallest normal), and fp32 noise of the
    pair's magnitude."""
    u = UNIT[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == F16 else 0.0
    err = (got.double() - want).abs()
    noise = 4e-6 * want.abs().amax(-1, keepdim=True)
    assert (err <= u * want.abs() + tiny + noise).all(), float(err.max())


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(16, 16, 128), (32, 8, 128), (14, 2, 64), (1, 1, 64), (64, 8, 128), (128, 8, 128)])
@pytest.mark.parametrize("norm,theta", [(True, 1e4), (False, 5e5), (True, None), (False, None)])
def test_append(ops, act, cache, H, Hk, D, norm, theta):
    new, kv, page = [1, 7, 0, 40], [1, 300, 4, 70000], 16
    rows = sum(new)
    k, v, table = make_cache(kv, Hk, D, page, cache)
    k0, v0 = k.clone(), v.clone()
    g = torch.Generator().manual_seed(7)
    qkv = (torch.randn(rows, (H + 2 * Hk) * D + 8, generator=g) * 3).to(act).cuda()[:, : (H + 2 * Hk) * D]
    qn = (1 + 0.2 * torch.randn(H * D, generator=g)).to(F16).cuda() if norm else None
    kn = (1 + 0.2 * torch.randn(Hk * D, generator=g)).to(F16).cuda() if norm else None
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    want_pos = torch.cat([torch.arange(L - n, L) for n, L in zip(new, kv)])
    assert torch.equal(plan.positions.cpu().long(), want_pos)
    assert plan.requests.cpu().tolist() == [r for r, n in enumerate(new) for _ in range(n)]
    q = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H, q_norm=qn, k_norm=kn, rope_theta=theta)
    wq, wk, wv = append_reference(qkv, H, Hk, D, plan.positions, qn, kn, 1e-5, theta)
    near(q, wq)
    pos, req = plan.positions.long(), plan.requests.long()
    ids = table[req, pos // page].long()
    near(k[ids, :, pos % page], wk)
    near(v[ids, :, pos % page], wv)
    k0[ids, :, pos % page] = k[ids, :, pos % page]
    v0[ids, :, pos % page] = v[ids, :, pos % page]
    assert torch.equal(k, k0) and torch.equal(v, v0), "another slot was written"


def test_append_skips_slots_that_do_not_exist(ops):
    """Positions before 0 or past the table, requests and page ids out of range: nothing is stored, q still comes."""
    H = Hk = 2
    D, page = 64, 16
    k, v, table = make_cache([32, 32], Hk, D, page, F16)
    k0, v0 = k.clone(), v.clone()
    table[1, 1] = -1
    table[1, 0] = k.shape[0]
    pos = torch.tensor([-1, 32, 2 ** 31 - 1, 0, 0, 20, 3], dtype=torch.int32, device="cuda")
    req = torch.tensor([0, 0, 0, 2, -1, 1, 1], dtype=torch.int32, device="cuda")
    qkv = torch.randn(7, 3 * H * D, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    q = ops.paged_append(qkv, k, v, table, pos, req, H)
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    assert torch.equal(q.reshape(7, -1), qkv[:, : H * D])


def test_append_then_attend_matches_contiguous_decode(ops):
    """One decode step equals the contiguous-cache operator on the same history."""
    B, H, D, cap, page = 3, 16, 128, 512, 64
    lens = [1, 200, 511]
    g = torch.Generator().manual_seed(11)
    kc = torch.randn(B, H, cap, D, generator=g).to(F16).cuda()
    vc = torch.randn(B, H, cap, D, generator=g).to(F16).cuda()
    qkv = torch.randn(B, 3 * H * D, generator=g).to(F16).cuda()
    qn = (1 + 0.1 * torch.randn(H * D, generator=g)).to(F16).cuda()
    kn = (1 + 0.1 * torch.randn(H * D, generator=g)).to(F16).cuda()
    table = torch.randperm(B * cap // page, generator=g).to(torch.int32).view(B, -1).cuda()
    k = torch.empty(B * cap // page, H, page, D, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    k[table.long()] = kc.view(B, H, -1, page, D).transpose(1, 2)
    v[table.long()] = vc.view(B, H, -1, page, D).transpose(1, 2)
    plan = ops.PagedPlan([1] * B, lens, H, H, D, page)
    q = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H, q_norm=qn, k_norm=kn, rope_theta=1e4)
    got = ops.paged_attention(q, k, v, table, plan).view(B, -1)
    want = ops.attention_decode(qkv, qn, kn, plan.positions, kc, vc, 1e-5, 1e4)
    # Both sides round q, k, p and the output to f16; |v| < 5.
    assert (got.double() - want.double()).abs().max() <= 4 * 5 * UNIT[F16]


# ---------------------------------------------------------------- refusals


def test_refusals(ops):
    k, v, table = make_cache([40, 40], 2, 64, 16, F16)
    plan = ops.PagedPlan([1, 1], [40, 40], 4, 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=F16, device="cuda")

    def bad(error, call, *a, **kw):
        with pytest.raises(error):
            call(*a, **kw)

    from trifuse_b200 import TriFuseError
    att = ops.paged_attention
    bad(ValueError, att, q[:1], k, v, table, plan)                       # rows differ from the plan
    bad(ValueError, att, q, k, v[:, :, :8], table, plan)                 # k and v differ
    bad(ValueError, att, q, k.transpose(1, 2), v.transpose(1, 2), table, plan)
    bad(ValueError, att, q, k, v, table.long(), plan)
    bad(ValueError, att, q, k, v, table[:1], plan)                       # fewer requests than planned
    bad(ValueError, att, q, k, v, table[:, :1], plan)                    # fewer pages than planned
    bad(ValueError, att, q.cpu(), k, v, table, plan)
    bad(ValueError, att, q.float(), k, v, table, plan)
    bad(ValueError, att, q, k.float(), v.float(), table, plan)
    bad(TriFuseError, att, q, k.bfloat16(), v.bfloat16(), table, plan)   # f16 queries over a bf16 cache
    bad(ValueError, att, q, k, v, table, plan, scale=0.0)
    bad(ValueError, att, q, k, v, table, plan, scale=float("nan"))
    bad(ValueError, att, q, k, v, table, plan, out=torch.empty(2, 4, 64, device="cuda"))
    other = ops.PagedPlan([1, 1], [40, 40], 4, 2, 64, 32)
    bad(ValueError, att, q, k, v, table, other)                          # planned for another page size
    qkv = torch.zeros(2, 8 * 64, dtype=F16, device="cuda")
    app = ops.paged_append
    pos, req = plan.positions, plan.requests
    bad(ValueError, app, qkv[:, :-64], k, v, table, pos, req, 4)
    bad(ValueError, app, qkv, k, v, table, pos[:1], req, 4)
    bad(ValueError, app, qkv, k, v, table, pos.long(), req, 4)
    bad(ValueError, app, qkv, k, v, table, pos, req, 4, q_norm=torch.ones(256, dtype=F16, device="cuda"))
    bad(ValueError, app, qkv, k, v, table, pos, req, 4, rope_theta=0.5)
    bad(ValueError, app, qkv, k, v, table, pos, req, 3)
