"""8-bit paged attention is off by what it rounds: weights once, outputs once.  (A second rounding of the weights, or
codes or scales rounded on their way, would show.)"""
import pytest
import torch

from tests.paged8_bounds import Exact, check_rounding
from tests.paged8_util import BF16, E4M3, F16, I8, Cache

pytestmark = pytest.mark.gpu

KINDS = [I8, E4M3]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def run(ops, new, kv, H, Hk, D, page, act, kind, size=2.0, seed=0, **kw):
    c = Cache(kv, Hk, D, page, kind, seed=seed + len(kv))
    q = (torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(seed + 1)) * size).to(act).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, new, kv), **kw)


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [0.3, 2.0])
@pytest.mark.parametrize("H,Hk,D,page,new,kv", [
    (16, 16, 128, 16, [1] * 9, [1, 2, 15, 16, 17, 32, 33, 600, 5003]), (8, 1, 64, 64, [1] * 5, [40, 333, 9000, 31, 64]),
    (14, 2, 64, 32, [1, 2, 1], [700, 900, 3000]), (8, 2, 128, 16, [4, 3], [900, 20]), (4, 2, 128, 16, [40, 60], [900, 61]),
    (32, 8, 128, 16, [130, 7, 257], [130, 500, 1300]), (6, 6, 64, 256, [300, 1, 129], [2049, 1, 129]), (2, 2, 128, 64, [40], [20000])])
def test_ordinary_calls(ops, act, kind, size, H, Hk, D, page, new, kv):
    run(ops, new, kv, H, Hk, D, page, act, kind, size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,Hk,D,new,kv", [(16, 16, 128, [1] * 40, list(range(2, 42))), (8, 2, 64, [2] * 30, list(range(3, 33))),
                                           (4, 4, 128, [16] * 6, [20, 16, 30, 25, 31, 17]), (4, 2, 128, [40, 50], [100, 128]),
                                           (8, 2, 64, [60, 100], [120, 100])])
def test_a_dominant_key_is_not_rounded(ops, kind, H, Hk, D, new, kv):
    """f16 outputs that one key makes up, whose block's scale is not the largest: its weight is a power of two, so what is
    left is the output's rounding and the other keys'.  (Histories of a tile: the many-rows kernel raises its reference
    with the first tile, later ones only by steps of 2^7.)"""
    run(ops, new, kv, H, Hk, D, 16, F16, kind, size=8.0, largest_exact=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,n,G", [(24, 5, 32), (40, 140, 1)])
def test_many_requests_on_one_prompt(ops, kind, B, n, G):
    """Requests that share their pages, each with more than 128 packed rows: the scratch holds the history once for each
    of them."""
    L, page, D = 1500, 16, 128
    c = Cache([L], 1, D, page, kind, seed=n)
    c.table = c.table.expand(B, -1).contiguous()
    q = (torch.randn(B * n, G, D, generator=torch.Generator().manual_seed(1)) * 2).to(BF16).cuda()
    plan = ops.PagedPlan([n] * B, [L] * B, G, 1, D, page)
    pages = -(-L // page)
    assert plan.widened_bytes >= 2 * B * pages * page * (2 * D + 4 // 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n] * B, [L] * B))
