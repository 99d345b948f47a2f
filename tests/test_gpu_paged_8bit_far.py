"""The 8-bit cache where numbers, shapes or tables are unusual: scores of 10^8, many small weights, pages that do not
exist, wide groups, replayed appends."""
import math

import pytest
import torch

from tests.paged8_util import BF16, BLOCK, E4M3, F16, I8, LARGEST, UNIT, Cache, attend, check

pytestmark = pytest.mark.gpu

KINDS = [I8, E4M3]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [300.0, 7000.0, 40000.0])
@pytest.mark.parametrize("n,L", [(1, 3000), (5, 700), (40, 3000), (130, 130), (300, 2500)])
@pytest.mark.parametrize("order", ["rising", "falling", "negative", "mixed"])
def test_far_scores(ops, act, kind, size, n, L, order):
    """Keys of one direction, a block of tokens each, in steps of 3 per cent: the largest score decides (with those equal
    to it), by millions."""
    H, Hk, D, page = 4, 2, 64, 16
    c = Cache([L], Hk, D, page, kind, seed=n)
    block = torch.arange(-(-L // BLOCK))
    step = {"rising": block // 6, "falling": (len(block) - block) // 6, "negative": block // 6,
            "mixed": (block * 7919) % 29}[order]
    c.k[c.table[0].long()] = int(LARGEST[kind]) if kind == I8 else torch.tensor(448.0, device="cuda").to(kind)
    c.ks[c.table[0].long(), :, 0] = (size * 1.03 ** (step.double() % 40 - 40) / LARGEST[kind]).float().cuda()[:, None]
    g = torch.Generator().manual_seed(n)
    q = (size * (0.5 + torch.rand(n, H, 1, generator=g))).to(act).expand(n, H, D).contiguous().cuda()
    if order == "negative":
        q.neg_()
    plan = ops.PagedPlan([n], [L], H, Hk, D, page)
    got = ops.paged_attention(q, *c.args(), plan, scale=1.0, **c.scales())
    assert ops.device_error() == 0
    want, big, _ = attend(c, q, [n], [L], 1.0)
    check(got, want, big, torch.zeros_like(big))  # one direction: no rounding of a key moves them apart


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gap", [9.0, 12.0, 15.0, 17.47])
@pytest.mark.parametrize("B,n,G,L,D,sinks", [(1, 200, 1, 60000, 64, [0]), (1, 20, 2, 60000, 128, [0]), (3, 300, 1, 40000, 128, [0, 7]),
                                             (1, 1, 1, 60000, 64, [0]), (148, 4, 4, 100000, 64, [0, 32, 64, 96])])
def test_many_small_weights_count(ops, act, kind, gap, B, n, G, L, D, sinks):
    """Scores 0 but for the sinks' gap; values 0 at the sinks, about 1 elsewhere: an output is the others' share.  Weights
    keep their 11 bits down to 2^-20 of the largest (the value scale over its power of two may cost one bit)."""
    page = 256
    pages = -(-L // page)
    largest = LARGEST[kind]
    k = torch.zeros(pages, 1, page, D, device="cuda")
    v = torch.full_like(k, largest)
    v[..., 1::2] = 0.75 * largest if kind == E4M3 else 95.0
    ks, vs = (torch.full((pages, 1, page // BLOCK), 1 / largest, device="cuda") for _ in range(2))
    for s in sinks:
        k[s // page, 0, s % page, 0] = largest
        v[s // page, 0, s % page] = 0
        ks[s // page, 0, s % page // BLOCK] = gap / largest
    k8, v8 = k.to(kind), v.to(kind)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].repeat(B, 1)  # the requests share their pages
    q = torch.zeros(B * n, G, D, dtype=act, device="cuda")
    q[..., 0] = 1
    plan = ops.PagedPlan([n] * B, [L] * B, G, 1, D, page)
    got = ops.paged_attention(q, k8, v8, table, plan, scale=1.0, k_scales=ks, v_scales=vs).double()
    assert ops.device_error() == 0
    others = torch.arange(L - n + 1, L + 1, dtype=torch.float64, device="cuda") - len(sinks)
    mass = others * math.exp(-gap)
    want = (mass / (mass + len(sinks))).repeat(B)[:, None, None] * (v8[-1, 0, 0].double() / largest)
    err = (got - want).abs()
    bound = UNIT[F16] + UNIT[act] * want + 1e-4 + 1e-6
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,G", [(1, 2), (3, 4), (40, 1), (300, 2)])
def test_pages_that_do_not_exist(ops, kind, n, G):
    """Ids below 0 and past the cache inside a history read as keys and values of zero."""
    L, Hk, D, page = 700, 2, 64, 32
    c = Cache([L], Hk, D, page, kind)
    q = torch.randn(n, G * Hk, D, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    plan = ops.PagedPlan([n], [L], G * Hk, Hk, D, page)
    zeros = Cache([L], Hk, D, page, kind)
    for i, bad in ((0, -1), (3, c.k.shape[0]), (4, 2 ** 31 - 1), (9, -2 ** 31)):
        at = zeros.table[0, i].long()
        for codes, scales in ((zeros.k, zeros.ks), (zeros.v, zeros.vs)):
            codes[at] = 0
            scales[at] = 0
        c.table[0, i] = bad
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check(got, *attend(zeros, q, [n], [L]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hk,D", [(32, 1, 128), (64, 2, 64), (128, 1, 128), (256, 1, 64), (200, 1, 64)])
def test_wide_groups(ops, kind, H, Hk, D):
    """Single tokens whose query heads alone fill the tensor-core kernels."""
    kv = [1, 16, 333, 4001]
    c = Cache(kv, Hk, D, 16, kind)
    q = (torch.randn(len(kv), H, D, generator=torch.Generator().manual_seed(1)) * 2).to(BF16).cuda()
    plan = ops.PagedPlan([1] * len(kv), kv, H, Hk, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check(got, *attend(c, q, [1] * len(kv), kv))


@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_append_follows_its_positions(ops, kind):
    """One graph, replayed at other positions of other requests: what the calls one by one store."""
    H, Hk, D, page, R = 4, 2, 64, 16, 5
    g = torch.Generator().manual_seed(2)
    a, b = (Cache([64] * R, Hk, D, page, kind, seed=4) for _ in range(2))
    qkv = torch.randn(8, (H + 2 * Hk) * D, generator=g).to(F16).cuda()
    pos, req = (torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.zeros(8, H, D, dtype=F16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.paged_append(qkv, *a.args(), pos, req, H, rope_theta=1e4, out=out, **a.scales())
    for p, r in (([0, 1, 2, 3, 4, 5, 6, 7], [0] * 8), ([8, 15, 16, 17, 0, 40, 41, 42], [0, 0, 0, 0, 1, 2, 2, 2]),
                 ([9, 1, 43, 31, 32, 33, 5, 6], [0, 1, 2, 3, 3, 3, 4, 4])):
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        req.copy_(torch.tensor(r, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(F16))
        graph.replay()
        torch.cuda.synchronize()
        q = ops.paged_append(qkv, *b.args(), pos, req, H, rope_theta=1e4, **b.scales())
        assert torch.equal(q, out)
        for x, y in zip((a.k, a.v, a.ks, a.vs), (b.k, b.v, b.ks, b.vs)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_an_empty_append(ops):
    c = Cache([40], 2, 64, 16, I8)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    q = ops.paged_append(torch.zeros(0, 8 * 64, dtype=F16, device="cuda"), *c.args(), none, none, 4, **c.scales())
    assert q.shape == (0, 4, 64)
