"""Append to and attention over a paged cache of 8-bit codes, against their formulas in 64 bits."""
import pytest
import torch

from tests.paged8_util import BF16, BLOCK, E4M3, F16, I8, LARGEST, UNIT, Cache, attend, check
from tests.test_gpu_paged import append_reference, near

pytestmark = pytest.mark.gpu

KINDS = [I8, E4M3]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def run(ops, new, kv, H, Hk, D, page, act, kind, seed=0, scale=None, **cache):
    c = Cache(kv, Hk, D, page, kind, seed, **cache)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(sum(new), H, D, generator=g) * 2).to(act).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    got = ops.paged_attention(q, *c.args(), plan, scale=scale, **c.scales())
    assert ops.device_error() == 0 and got.dtype == act
    check(got, *attend(c, q, new, kv, scale))
    return c, q, plan, got


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(16, 16), (8, 1), (14, 2), (6, 2)])
def test_decode(ops, act, kind, D, H, Hk):
    """Single tokens, from one key to several splits, lengths around block, tile and page ends."""
    run(ops, [1] * 9, [1, 2, 15, 16, 17, 32, 33, 600, 5003], H, Hk, D, 16, act, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes(ops, kind, page):
    run(ops, [1, 3, 1, 2, 40, 300], [7, 300, 257, 1025, 555, 999], 8, 2, 128, page, BF16, kind)


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,H,Hk", [(128, 16, 16), (64, 14, 2), (128, 32, 8), (128, 5, 1), (64, 6, 6)])
def test_chunks(ops, act, kind, D, H, Hk):
    """Chunks of many lengths in one call: whole prompts, late chunks, single tokens, an idle request."""
    run(ops, [1, 130, 0, 257, 1, 77, 300], [900, 130, 50, 1300, 1, 500, 2049], H, Hk, D, 16, act, kind)


@pytest.mark.parametrize("n", [1, 2, 16, 17, 33, 64, 127, 128, 129, 255, 256, 257, 511])
def test_prompt_lengths(ops, n):
    run(ops, [n], [n], 4, 2, 128, 32, F16, KINDS[n % 2], seed=n)


@pytest.mark.parametrize("n,L", [(1, 127), (1, 129), (5, 4096), (40, 4097), (64, 8191), (300, 20000)])
def test_long_history(ops, n, L):
    """Few rows over a long history: the keys are divided and the parts merged."""
    run(ops, [n], [L], 8, 2, 128, 64, BF16, KINDS[L % 2], seed=L)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 40, 300])
def test_scales_far_apart(ops, kind, n):
    """Blocks whose magnitudes differ by up to 2^20: the references move often."""
    run(ops, [n, n], [900, 2000], 4, 2, 128, 16, F16, kind, seed=n, spread=20, scale=0.01)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 40, 300])
def test_zero_scales(ops, kind, n):
    """Blocks of nothing but zeros, and caches of them."""
    L = 700
    c = Cache([L], 2, 128, 16, kind)
    q = torch.randn(n, 4, 128, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    plan = ops.PagedPlan([n], [L], 4, 2, 128, 16)
    for pages in (slice(0, None, 3), slice(None)):
        for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
            codes[pages] = 0
            scales[pages] = 0
        got = ops.paged_attention(q, *c.args(), plan, **c.scales())
        check(got, *attend(c, q, [n], [L]))
    assert (got == 0).all()


def test_rows_that_attend_nothing(ops):
    """kv shorter than the new tokens: the rows before token 0 give zeros; so does an empty history."""
    for new, kv in (([5], [3]), ([1, 4], [0, 0]), ([40, 300], [30, 0]), ([200], [70])):
        *_, got = run(ops, new, kv, 8, 2, 128, 16, F16, I8)
        assert (got[: max(0, new[0] - kv[0])] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hk,D,n,L", [(4, 4, 64, 2, 20), (4, 4, 128, 16, 700), (8, 2, 64, 4, 5000), (4, 2, 128, 40, 700),
                                        (2, 2, 64, 128, 9000), (4, 4, 128, 300, 300), (4, 1, 128, 150, 6000)])
def test_nan_scales(ops, kind, H, Hk, D, n, L):
    """A NaN scale of keys or values reaches the rows that see a token of its block, and nothing else changes by a
    bit."""
    G, page = H // Hk, 16
    c = Cache([L, L], Hk, D, page, kind)
    q = torch.randn(2 * n, H, D, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    plan = ops.PagedPlan([n, n], [L, L], H, Hk, D, page)
    clean = ops.paged_attention(q, *c.args(), plan, **c.scales())
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for r, t, h, scales in ((0, L - 1, 0, c.vs), (1, L - 1 - n // 2, Hk - 1, c.ks), (1, L - n // 4 - 1, 0, c.vs)):
        scales[c.table[r, t // page].long(), h, t % page // BLOCK] = float("nan")
        first = n * r + max(0, t // BLOCK * BLOCK - (L - n))
        hit[first:n * (r + 1), h * G:(h + 1) * G] = True
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    assert torch.isfinite(clean).all() and torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("n", [1, 60])
def test_strides_and_interleaved_pages(ops, n):
    """q as a slice of a fused projection, k and v pages and their scales in one buffer each, a wide page table."""
    H, Hk, D, page, L = 8, 2, 128, 32, 333
    c = Cache([L, L], Hk, D, page, I8)
    both = torch.full((c.k.shape[0], 2, Hk, page, D), 0x81 - 256, dtype=I8, device="cuda")
    both[:, 0], both[:, 1] = c.k, c.v
    scales = torch.full((c.k.shape[0], 2, Hk, page // BLOCK), float("nan"), device="cuda")
    scales[:, 0], scales[:, 1] = c.ks, c.vs
    wide = torch.full((2, c.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + c.table.shape[1]] = c.table
    fused = torch.randn(2 * n, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(5)).to(F16).cuda()
    q = fused[:, : H * D].view(2 * n, H, D)
    plan = ops.PagedPlan([n, n], [L, L], H, Hk, D, page)
    want = ops.paged_attention(q.contiguous(), *c.args(), plan, **c.scales())
    out = torch.empty_like(want)
    got = ops.paged_attention(q, both[:, 0], both[:, 1], wide[:, 2:2 + c.table.shape[1]], plan, out=out,
                              k_scales=scales[:, 0], v_scales=scales[:, 1])
    assert got is out and torch.equal(got, want)


def test_repeatable_other_stream_and_captured(ops):
    """The same plan gives the same bits again, on another stream and from a graph; it serves a 16-bit cache beside."""
    new, kv = [1, 30, 300, 1], [9000, 4000, 5000, 17]
    c, q, plan, got = run(ops, new, kv, 8, 2, 128, 16, BF16, E4M3)
    half = [torch.randn(c.k.shape, dtype=BF16, device="cuda") for _ in range(2)]
    other = ops.paged_attention(q, *half, c.table, plan)
    for _ in range(20):
        assert torch.equal(ops.paged_attention(q, *c.args(), plan, **c.scales()), got)
    assert torch.equal(ops.paged_attention(q, *half, c.table, plan), other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.paged_attention(q, *c.args(), plan, **c.scales())
    side.synchronize()
    assert torch.equal(again, got)
    out = torch.zeros_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.paged_attention(q, *c.args(), plan, out=out, **c.scales())
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_pages_beyond_four_gigabytes(ops):
    """Byte offsets past 32 bits in codes: used pages are the last of a cache of over 4 GB a side."""
    pages, Hk, page, D = 18000, 16, 128, 128  # 4.7 GB a side
    k = torch.zeros(pages, Hk, page, D, dtype=I8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(pages, Hk, page // BLOCK, device="cuda") for _ in range(2))
    L = 700
    table = torch.arange(pages - 6, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    qkv = torch.randn(L, 3 * Hk * D, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    small = Cache([L], Hk, D, page, I8)
    for new in ([L], [1]):
        plan = ops.PagedPlan(new, [L], Hk, Hk, D, page)
        n = new[0]
        q = ops.paged_append(qkv[:n], k, v, table, plan.positions, plan.requests, Hk, k_scales=ks, v_scales=vs)
        ids = table[0].long()
        at = small.table[0, :6].long()
        for a, b in ((small.k, k), (small.v, v), (small.ks, ks), (small.vs, vs)):
            a[at] = b[ids]
        got = ops.paged_attention(q, k, v, table, plan, k_scales=ks, v_scales=vs)
        check(got, *attend(small, q, new, [L]))
    assert (k[0] == 0).all() and (ks[0] == 0).all()


# ---------------------------------------------------------------- append


def append_check(c, before, want, lens, start):
    """Codes, scales and everything beside them after the tokens [start[r], lens[r]) of the requests were written.
    before: clones of k, v, ks, vs; want: k and v of the new rows [rows, Hk, D] in 64 bits."""
    page, kind, table = c.page, c.kind, c.table.tolist()
    for n, i in (("k", 0), ("v", 1)):
        codes, scales = getattr(c, n).cpu(), getattr(c, n + "s").cpu()
        old_codes, old_scales, x = before[i].cpu(), before[2 + i].cpu(), want[i].cpu()
        left, kept = codes.view(torch.uint8).clone(), scales.clone()
        row = 0
        for r, (a, b) in enumerate(zip(start, lens)):
            p = a
            while p < b:
                end = min(b, p // BLOCK * BLOCK + BLOCK)
                id, blk, slot = table[r][p // page], p % page // BLOCK, p % page
                new = x[row:row + end - p].transpose(0, 1)  # [Hk, tokens, D]
                amax = new.abs().amax((1, 2))
                s = amax / LARGEST[kind]
                held = slot % BLOCK
                if held:
                    s = torch.maximum(s, old_scales[id, :, blk].double())
                got_s = scales[id, :, blk].double()
                # fp32 noise of the norm and the rotation, one division.
                assert ((got_s - s).abs() <= 1e-5 * s).all()
                at = got_s[:, None, None]
                step = lambda y: 0.5001 if kind == I8 else torch.maximum(y.abs() * (2.0 ** -4 * 1.0001),  # noqa: E731
                                                                         torch.full_like(y, 2.0 ** -10 * 1.0001))
                y = new / at
                noise = 4e-6 * new.abs().amax(-1, keepdim=True) / at
                got = codes[id, :, slot:slot + end - p].float().double()
                assert ((got - y).abs() <= step(y) + noise).all()
                if held:
                    first = slot - held
                    o = old_codes[id, :, first:slot].float().double()
                    ratio = old_scales[id, :, blk].double()[:, None, None] / at
                    now = codes[id, :, first:slot].float().double()
                    grown = (got_s > old_scales[id, :, blk].double())[:, None, None]
                    assert ((now - o * ratio).abs() <= torch.where(grown, torch.as_tensor(step(o * ratio)).to(o), 0)).all()
                    left[id, :, first:slot] = old_codes.view(torch.uint8)[id, :, first:slot]
                left[id, :, slot:slot + end - p] = old_codes.view(torch.uint8)[id, :, slot:slot + end - p]
                kept[id, :, blk] = old_scales[id, :, blk]
                row += end - p
                p = end
        assert torch.equal(left, old_codes.view(torch.uint8)), "another slot was written"
        assert torch.equal(kept.view(torch.int32), old_scales.view(torch.int32)), "another scale was written"


def clones(c):
    return [getattr(c, n).clone() for n in ("k", "v", "ks", "vs")]


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hk,D,norm,theta", [(16, 16, 128, True, 1e4), (32, 8, 128, False, 5e5), (14, 2, 64, True, None),
                                               (1, 1, 64, False, None), (80, 40, 128, True, 1e4),
                                               (128, 8, 128, False, 1e4)])
def test_append(ops, act, kind, H, Hk, D, norm, theta):
    new, kv, page = [1, 7, 0, 40, 1, 16, 33], [1, 300, 4, 70000, 31, 64, 50], 32
    rows = sum(new)
    c = Cache(kv, Hk, D, page, kind, spread=6)
    before = clones(c)
    g = torch.Generator().manual_seed(7)
    qkv = (torch.randn(rows, (H + 2 * Hk) * D + 8, generator=g) * 1.5).to(act).cuda()[:, : (H + 2 * Hk) * D]
    qn = (1 + 0.2 * torch.randn(H * D, generator=g)).to(F16).cuda() if norm else None
    kn = (1 + 0.2 * torch.randn(Hk * D, generator=g)).to(F16).cuda() if norm else None
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    q = ops.paged_append(qkv, *c.args(), plan.positions, plan.requests, H, q_norm=qn, k_norm=kn, rope_theta=theta,
                         **c.scales())
    wq, wk, wv = append_reference(qkv, H, Hk, D, plan.positions, qn, kn, 1e-5, theta)
    near(q, wq)
    append_check(c, before, (wk, wv), kv, [b - a for a, b in zip(new, kv)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[900], [799, 1, 30], [1] * 900, [3] * 400, [17] * 60])
def test_append_many_rows(ops, kind, new):
    """Windows of 16 rows: units that begin at any place of them, several in one."""
    kv = [n + 5 + 3 * i % 40 for i, n in enumerate(new)]
    H, Hk, D, page = 4, 2, 64, 16
    c = Cache(kv, Hk, D, page, kind)
    before = clones(c)
    qkv = torch.randn(sum(new), (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(7)).to(F16).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    q = ops.paged_append(qkv, *c.args(), plan.positions, plan.requests, H, rope_theta=1e4, **c.scales())
    wq, wk, wv = append_reference(qkv, H, Hk, D, plan.positions, None, None, 1e-5, 1e4)
    near(q, wq)
    append_check(c, before, (wk, wv), kv, [b - a for a, b in zip(new, kv)])


@pytest.mark.parametrize("kind", KINDS)
def test_append_token_by_token(ops, kind):
    """One token at a time over two blocks: each scale is the largest so far, and what is held stays within a step of
    the token (a code that is rounded anew at each rise of the scale is off by half a step each time)."""
    H, Hk, D, page, L = 2, 2, 64, 16, 37
    c = Cache([L], Hk, D, page, kind)
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(L, 3 * Hk * D, generator=g) * (1 + torch.arange(L)[:, None] % 5)).to(F16).cuda()
    for t in range(L):
        before = clones(c)
        pos = torch.tensor([t], dtype=torch.int32, device="cuda")
        ops.paged_append(x[t:t + 1], *c.args(), pos, torch.zeros_like(pos), H, **c.scales())
        k, v = (x[t:t + 1, (1 + i) * Hk * D:(2 + i) * Hk * D].double().view(1, Hk, D) for i in range(2))
        append_check(c, before, (k, v), [t + 1], [t])


@pytest.mark.parametrize("kind", KINDS)
def test_append_values_at_the_ends(ops, kind):
    """Zeros, the type's smallest and largest values, and NaN or infinities, each in a head of its own."""
    H, Hk, D, page = 6, 6, 64, 16
    c = Cache([20], Hk, D, page, kind)
    x = torch.randn(4, Hk, D, generator=torch.Generator().manual_seed(5)).to(BF16)
    x[:, 0] = 0
    x[:, 1] = 9.2e-41
    x[:, 2] *= 1e-39
    x[:, 3, 7] = 3.38e38
    x[2, 4, 3] = float("nan")
    x[1, 5, 60] = float("inf")
    qkv = torch.cat([torch.zeros(4, H * D, dtype=BF16), x.flatten(1), x.flatten(1)], 1).cuda()
    pos = torch.arange(16, 20, dtype=torch.int32, device="cuda")
    ops.paged_append(qkv, *c.args(), pos, torch.zeros_like(pos), H, **c.scales())
    page1 = int(c.table[0, 1])
    for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
        s = scales[page1, :, 0]
        assert s[0] == 0 and (codes[page1, 0, :4].float() == 0).all()
        assert s[1] == s[2] == 2.0 ** -126
        got = codes[page1, 1:4, :4].float().double() * s[1:4].double()[:, None, None]
        want = x[:, 1:4].double().transpose(0, 1).cuda()
        step = s[1:4].double()[:, None, None] * (0.5001 if kind == I8 else 2.0 ** -10)
        assert ((got - want).abs() <= step + (0 if kind == I8 else 2.0 ** -4 * 1.0001) * want.abs()).all()
        assert torch.isnan(s[4:]).all() and torch.isfinite(codes[page1].float()[:, :4]).all()
    # The next token of the block finds its scale; a block that is begun anew does not.
    ops.paged_append(torch.ones_like(qkv[:1]), *c.args(), pos[:1] + 4, torch.zeros_like(pos[:1]), H, **c.scales())
    assert torch.isnan(c.ks[page1, 4:, 0]).all() and torch.isfinite(c.ks[page1, :4, 0]).all()
    ops.paged_append(torch.ones_like(qkv[:1]), *c.args(), pos[:1], torch.zeros_like(pos[:1]), H, **c.scales())
    assert torch.allclose(c.ks[page1, :, 0], torch.full((Hk,), 1 / LARGEST[kind], device="cuda"), rtol=1e-6)


def test_append_skips_slots_that_do_not_exist(ops):
    """Positions before 0 or past the table, requests and page ids out of range: nothing is stored, q still comes."""
    H = Hk = 2
    D, page = 64, 16
    c = Cache([32, 32], Hk, D, page, I8)
    before = clones(c)
    c.table[1, 1] = -1
    c.table[1, 0] = c.k.shape[0]
    pos = torch.tensor([-1, 32, 2 ** 31 - 1, -2 ** 31, 0, 0, 20, 3], dtype=torch.int32, device="cuda")
    req = torch.tensor([0, 0, 0, 0, 2, -1, 1, 1], dtype=torch.int32, device="cuda")
    qkv = torch.randn(8, 3 * H * D, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    q = ops.paged_append(qkv, *c.args(), pos, req, H, **c.scales())
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, clones(c)))
    assert torch.equal(q.reshape(8, -1), qkv[:, : H * D])


def test_append_then_attend(ops):
    """Chunk after chunk and token after token into one cache, attended each time: near attention over the 16-bit
    values.  Keys are off by 1/254 (int8) of their block's largest magnitude at most; with scores of standard deviation
    one the output's norm moves by less than 5 per cent."""
    H, Hk, D, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(2)
    total = 150
    qkv = torch.randn(total, (H + 2 * Hk) * D, generator=g).to(F16).cuda()
    for kind in KINDS:
        c = Cache([total], Hk, D, page, kind)
        k16, v16 = (torch.zeros(c.k.shape, dtype=F16, device="cuda") for _ in range(2))
        at = 0
        for n in (70, 1, 1, 1, 40, 3, 34):
            plan = ops.PagedPlan([n], [at + n], H, Hk, D, page)
            rows = qkv[at:at + n]
            q = ops.paged_append(rows, *c.args(), plan.positions, plan.requests, H, rope_theta=1e4, **c.scales())
            q16 = ops.paged_append(rows, k16, v16, c.table, plan.positions, plan.requests, H, rope_theta=1e4)
            assert torch.equal(q, q16)
            got = ops.paged_attention(q, *c.args(), plan, **c.scales())
            want = ops.paged_attention(q, k16, v16, c.table, plan)
            check(got, *attend(c, q, [n], [at + n]))
            assert (got - want).float().norm() <= 0.05 * want.float().norm()
            at += n


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [16, 100])
@pytest.mark.parametrize("H,Hk,D,new,kv", [(4, 4, 128, [1, 1], [1, 700]), (14, 2, 64, [1, 2], [40, 9000]),
                                           (8, 2, 64, [9, 30], [5000, 30]), (4, 2, 128, [257, 64], [257, 4000])])
def test_queries_beyond_f16(ops, kind, power, H, Hk, D, new, kv):
    """bf16 queries past f16's range, all rows and every third one; the scale brings the scores back, so the bounds are
    those of ordinary ones."""
    c = Cache(kv, Hk, D, 16, kind, seed=3)
    plan = ops.PagedPlan(new, kv, H, Hk, D, 16)
    q = (torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(4)) * 2).to(BF16).cuda()
    some = q.clone()
    some[::3, ::2] *= 2.0 ** power
    scale = 2.0 ** -power * D ** -0.5
    for x in (q * 2.0 ** power, some):
        got = ops.paged_attention(x, *c.args(), plan, scale=scale, **c.scales())
        assert ops.device_error() == 0
        check(got, *attend(c, x, new, kv, scale), rms=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_an_infinite_query_stays_in_its_row(ops, kind, n):
    """NaN and infinite queries make their own (row, head) NaN and leave the others' bits."""
    H, Hk, D, L = 4, 2, 128, 700
    c = Cache([L], Hk, D, 16, kind)
    plan = ops.PagedPlan([n], [L], H, Hk, D, 16)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(n)).to(BF16).cuda()
    want = ops.paged_attention(q, *c.args(), plan, **c.scales())
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[n // 2, 1, 17] = bad
        got = ops.paged_attention(x, *c.args(), plan, **c.scales())
        assert torch.isnan(got[n // 2, 1]).all()
        got[n // 2, 1] = want[n // 2, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("L", [9000, 33000])
@pytest.mark.parametrize("H,Hk,D", [(1, 1, 64), (1, 1, 128), (7, 1, 64), (8, 1, 128), (12, 1, 128), (16, 1, 64)])
def test_many_pieces(ops, H, Hk, D, L):
    """One long request whose pieces lie on every SM: all ways to share them among threads."""
    run(ops, [1], [L], H, Hk, D, 64, F16, KINDS[H % 2], seed=H)


def test_refusals(ops):
    from trifuse_b200 import TriFuseError
    c = Cache([40], 2, 64, 16, I8)
    plan = ops.PagedPlan([1], [40], 4, 2, 64, 16)
    q = torch.zeros(1, 4, 64, dtype=F16, device="cuda")
    qkv = torch.zeros(1, 8 * 64, dtype=F16, device="cuda")
    before = [x.nan_to_num().clone() if x.is_floating_point() else x.clone() for x in (c.k, c.v, c.ks, c.vs)]
    pages16 = c.k.half()
    for k, v, ks, vs in ((c.k, c.v, None, None), (c.k, c.v, c.ks, None), (pages16, pages16, c.ks, c.vs),
                         (c.k, c.v, c.ks[:1], c.vs), (c.k, c.v, c.ks.cpu(), c.vs), (c.k, c.v, c.ks.half(), c.vs.half()),
                         (c.k, c.v.view(torch.float8_e4m3fn), c.ks, c.vs)):
        kw = {n: x for n, x in (("k_scales", ks), ("v_scales", vs)) if x is not None}
        with pytest.raises((ValueError, TriFuseError)):
            ops.paged_attention(q, k, v, c.table, plan, **kw)
        with pytest.raises((ValueError, TriFuseError)):
            ops.paged_append(qkv, k, v, c.table, plan.positions, plan.requests, 4, **kw)
    small = torch.zeros(4, 2, 8, 64, dtype=I8, device="cuda")  # pages below a block of tokens
    with pytest.raises((ValueError, TriFuseError)):
        ops.paged_append(qkv, small, small, c.table, plan.positions, plan.requests, 4,
                         k_scales=torch.zeros(4, 2, 0, device="cuda"), v_scales=torch.zeros(4, 2, 0, device="cuda"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.nan_to_num() if b.is_floating_point() else b)
               for a, b in zip(before, (c.k, c.v, c.ks, c.vs)))


@pytest.mark.parametrize("new,kv", [([1] * 5, [700, 3000, 17, 9000, 40]), ([30, 25], [3000, 900]), ([300], [5000]),
                                    ([1, 300, 40], [4000, 2000, 700])])
def test_waits_that_run_out(ops, new, kv):
    """With a limit of one cycle a wait that its first try does not meet runs out; the call ends all the same, and the
    next ones give what they gave."""
    from trifuse_b200._lib import check as ok, lib
    c, q, plan, want = run(ops, new, kv, 8, 2, 128, 16, BF16, E4M3)
    try:
        ok(lib().tf_set_wait_limit(1))
        for _ in range(3):
            ops.paged_attention(q, *c.args(), plan, **c.scales())
        torch.cuda.synchronize()
    finally:
        ok(lib().tf_set_wait_limit(0))
    assert ops.device_error() in (0, 71, *range(81, 96))
    for _ in range(3):
        assert torch.equal(ops.paged_attention(q, *c.args(), plan, **c.scales()), want)
    assert ops.device_error() == 0
