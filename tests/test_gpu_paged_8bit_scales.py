"""8-bit paged attention where the scales of values reach over fp32's range: values near bf16's largest, later tokens
that a row must not see, keys without weight beside keys with all of it, blocks of zeros."""
import math

import pytest
import torch

from tests.paged8_bounds import Exact, check_rounding
from tests.paged8_util import BF16, BLOCK, E4M3, F16, I8, LARGEST, Cache

pytestmark = pytest.mark.gpu

KINDS = [I8, E4M3]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def queries(rows, H, D, seed=1, act=BF16):
    return (torch.randn(rows, H, D, generator=torch.Generator().manual_seed(seed)) * 2).to(act).cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hk,D,new,kv", [(4, 4, 128, [1, 1], [700, 60000]), (4, 2, 64, [1] * 3, [1, 40, 20000]),
                                           (8, 2, 128, [4, 2], [9000, 333]), (4, 2, 128, [40, 60], [40, 20000]),
                                           (4, 2, 64, [64], [9000]), (2, 2, 128, [300, 130], [300, 20000])])
def test_values_near_the_types_largest(ops, kind, H, Hk, D, new, kv):
    """Values up to 1.7e38 (bf16 ends at 3.4e38), whole and in pieces."""
    c = Cache(kv, Hk, D, 16, kind, spread=0)
    real = ~torch.isnan(c.vs)
    c.vs *= 1.7e38 / (c.vs[real].max() * LARGEST[kind])
    q = queries(sum(new), H, D)
    plan = ops.PagedPlan(new, kv, H, Hk, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    ref = Exact(c, q, new, kv)
    check_rounding(got, ref)


def block_of(c, request, token):
    """Index of the token's block of scales."""
    return c.table[request, token // c.page].long(), slice(None), token % c.page // BLOCK


ROWS = [(1, 1, 657), (2, 2, 657), (5, 3, 657), (40, 2, 657), (300, 2, 657), (300, 1, 300), (1, 2, 20001), (40, 1, 20001)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [30, 70, 120])
@pytest.mark.parametrize("n,G,L", [(2, 2, 657), (5, 3, 657), (16, 1, 5009), (40, 2, 657), (40, 1, 20001), (130, 1, 657), (300, 2, 657),
                                   (300, 1, 305)])
def test_a_later_token_of_any_size(ops, kind, power, n, G, L):
    """The last token's block, and one in the middle of the new ones, hold values 2^power times as large: the rows before
    do not see them, and are as exact as without."""
    for token in {L - 1, L - n // 2}:
        c = Cache([L], 2, 128, 16, kind, seed=n, spread=1)
        c.vs[block_of(c, 0, token)] *= 2.0 ** power
        q = queries(n, 2 * G, 128, n)
        plan = ops.PagedPlan([n], [L], 2 * G, 2, 128, 16)
        got = ops.paged_attention(q, *c.args(), plan, **c.scales())
        assert ops.device_error() == 0
        ref = Exact(c, q, [n], [L])
        check_rounding(got, ref, scattered=False, exponents=2.0 ** -13)
        before = max(0, token // BLOCK * BLOCK - (L - n))
        if before:
            check_rounding(got[:before], ref.rows(slice(0, before)), exponents=2.0 ** -13)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [30, 100, 118])
@pytest.mark.parametrize("gap", [0.5, 20.0, 60.0, 88.0, 150.0, 300.0])
@pytest.mark.parametrize("blocks", [[0], [14, 15, 16, 17], [38, 39]])
@pytest.mark.parametrize("n,G,L", ROWS)
def test_large_values_of_little_weight(ops, kind, power, gap, blocks, n, G, L):
    """Blocks of e^-gap of the weight with values 2^power times as large: the first one, which every row sees, and
    several after others (tiles of nothing but such, a warp's first of the few-rows kernel and its second)."""
    D = 128
    c = Cache([L], 2, D, 16, kind, seed=n, spread=1)
    c.k[..., 0] = 0
    for block in (b for b in blocks if b < L // BLOCK):
        at = block_of(c, 0, block * BLOCK)
        c.k[at[0]] = 0  # pages of 16: one block
        c.k[at[0], ..., 0] = torch.tensor(-LARGEST[kind], device="cuda").to(kind)
        c.ks[at] = gap * D ** 0.5 / (4 * LARGEST[kind])
        c.vs[at] *= 2.0 ** power
    q = queries(n, 2 * G, D, n) * 0.5
    q[..., 0] = 4
    plan = ops.PagedPlan([n], [L], 2 * G, 2, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n], [L]), scattered=False, exponents=2.0 ** -13)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act,low,high", [(BF16, -110, 100), (BF16, -110, -50), (BF16, -60, 60), (F16, -110, 8)])
@pytest.mark.parametrize("size", [0.5, 4.0])
@pytest.mark.parametrize("n,G,L", ROWS + [(300, 2, 5000)])
def test_blocks_of_every_size(ops, kind, act, low, high, size, n, G, L):
    """Each block's values lie anywhere between 2^low and 2^high; every tenth block's scale is zero, whatever its codes."""
    c = Cache([L], 2, 64, 16, kind, seed=n, spread=0)
    g = torch.Generator().manual_seed(n + 1)
    power = torch.randint(low, high + 1, c.vs.shape, generator=g).cuda()
    c.vs *= torch.where((torch.rand(c.vs.shape, generator=g) < 0.1).cuda(), 0.0, 2.0 ** power)
    q = (torch.randn(n, 2 * G, 64, generator=g) * size).to(act).cuda()
    plan = ops.PagedPlan([n], [L], 2 * G, 2, 64, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n], [L]), scattered=False, exponents=2.0 ** -13)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [-116, -60, 60, 110])
@pytest.mark.parametrize("n,G,L", ROWS)
def test_all_values_large_or_small(ops, kind, power, n, G, L):
    """One power of two for all values: exact, so the outputs are those of ordinary ones."""
    c = Cache([L], 2, 128, 16, kind, seed=n)
    c.vs *= 2.0 ** power
    q = queries(n, 2 * G, 128, n)
    plan = ops.PagedPlan([n], [L], 2 * G, 2, 128, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n], [L]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [300.0, 7000.0, 40000.0])
@pytest.mark.parametrize("spread", [8, 16, 40, 200])
@pytest.mark.parametrize("n,L", [(1, 3000), (5, 700), (40, 3000), (300, 2500), (300, 300)])
def test_far_scores_of_blocks_of_every_size(ops, kind, size, spread, n, L):
    """Keys of one direction in steps of 3 per cent, scores to 10^9: the largest visible score decides, with those equal
    to it, whatever the other blocks' values."""
    H, Hk, D, page = 4, 2, 64, 16
    c = Cache([L], Hk, D, page, kind, seed=n, spread=0)
    g = torch.Generator().manual_seed(n)
    blocks = -(-L // BLOCK)
    step = torch.randint(0, 40, (blocks,), generator=g).double()
    ids = c.table[0].long()
    c.k[ids] = int(LARGEST[kind]) if kind == I8 else torch.tensor(448.0, device="cuda").to(kind)
    c.ks[ids, :, 0] = (size * 1.03 ** (step - 40) / LARGEST[kind]).float().cuda()[:, None]
    c.vs[ids, :, 0] = 2.0 ** (torch.randint(0, spread + 1, (blocks, 1), generator=g).float() - spread / 2).cuda()
    q = (size * (0.5 + torch.rand(n, H, 1, generator=g))).to(BF16).expand(n, H, D).contiguous().cuda()
    plan = ops.PagedPlan([n], [L], H, Hk, D, page)
    got = ops.paged_attention(q, *c.args(), plan, scale=1.0, **c.scales())
    assert ops.device_error() == 0
    ref = Exact(c, q, [n], [L], 1.0)
    ref.sums = torch.zeros_like(ref.sums)  # one direction: no rounding of a key moves them apart
    check_rounding(got, ref, scattered=False, exponents=2.0 ** -13)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,G,L", [(5, 3, 657), (40, 2, 657), (300, 2, 657), (300, 1, 300), (130, 2, 20001)])
def test_nan_scales_among_blocks_of_every_size(ops, kind, n, G, L):
    """A NaN scale of a value or a key makes the rows NaN that see its block; the others are as exact as without it."""
    c = Cache([L], 2, 64, 16, kind, seed=n, spread=0)
    g = torch.Generator().manual_seed(n + 1)
    c.vs *= (2.0 ** torch.randint(-100, 100, c.vs.shape, generator=g)).cuda()
    q = queries(n, 2 * G, 64, n)
    ref = Exact(c, q, [n], [L])
    plan = ops.PagedPlan([n], [L], 2 * G, 2, 64, 16)
    for scales, token in ((c.vs, L - 1), (c.ks, L - 1), (c.vs, L - n // 2)):
        at = block_of(c, 0, token)
        was = scales[at].clone()
        scales[at] = float("nan")
        got = ops.paged_attention(q, *c.args(), plan, **c.scales())
        assert ops.device_error() == 0
        scales[at] = was
        before = max(0, token // BLOCK * BLOCK - (L - n))
        assert torch.isnan(got[before:]).all()
        if before:
            check_rounding(got[:before], ref.rows(slice(0, before)), scattered=False, exponents=2.0 ** -13)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [30, 70, 118])
@pytest.mark.parametrize("gap", [20.0, 60.0, 150.0])
@pytest.mark.parametrize("n,G", [(1, 1), (4, 4)])
def test_scales_that_rise_within_a_warps_tiles(ops, kind, power, gap, n, G):
    """Requests enough that a block of warps has a whole history: each warp meets large values after small ones."""
    R, L, D = 80, 817, 128
    c = Cache([L] * R, 2, D, 16, kind, seed=n, spread=1)
    c.k[..., 0] = 0
    at = c.table[:, 26:50].long().flatten()  # the second tiles of the warps
    c.k[at] = 0
    c.k[at, ..., 0] = torch.tensor(-LARGEST[kind], device="cuda").to(kind)
    c.ks[at] = gap * D ** 0.5 / (4 * LARGEST[kind])
    c.vs[at] *= 2.0 ** power
    q = queries(R * n, 2 * G, D, n) * 0.5
    q[..., 0] = 4
    plan = ops.PagedPlan([n] * R, [L] * R, 2 * G, 2, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n] * R, [L] * R), scattered=False, exponents=2.0 ** -13)
