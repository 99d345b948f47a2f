"""Scores of 10^8 and beyond, which 16-bit queries and keys can make: the product with the scale is rounded there by
more than the exponential bears, so it must be the same rounding for the maximum and for each score."""
import pytest
import torch

from tests.test_gpu_paged import BF16, F16, TYPES, check, make_cache, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("size", [300.0, 2000.0, 7000.0, 40000.0])
@pytest.mark.parametrize("n,L", [(1, 3000), (5, 700), (40, 3000), (130, 130), (300, 2500)])
@pytest.mark.parametrize("order", ["rising", "falling", "negative", "mixed"])
def test_far_scores(act, cache, size, n, L, order):
    """Keys of one direction in steps of 3 per cent: the largest score decides (with those equal to it), by millions."""
    from trifuse_b200 import ops
    H, Hk, D, page = 4, 2, 64, 16
    k, v, table = make_cache([L], Hk, D, page, cache, seed=n)
    step = {"rising": torch.arange(L) // 100, "falling": (L - torch.arange(L)) // 100, "negative": torch.arange(L) // 100,
            "mixed": (torch.arange(L) * 7919) % 29}[order]
    rows = (size * 1.03 ** (step.double() % 40 - 40)).to(cache).cuda()
    for t in range(L):
        k[table[0, t // page].long(), :, t % page] = rows[t]
    g = torch.Generator().manual_seed(n)
    q = (size * (0.5 + torch.rand(n, H, 1, generator=g))).to(act).expand(n, H, D).contiguous().cuda()
    if order == "negative":
        q.neg_()
    plan = ops.PagedPlan([n], [L], H, Hk, D, page)
    got = ops.paged_attention(q, k, v, table, plan, scale=1.0)
    assert ops.device_error() == 0
    want, big = reference(q, k, v, table, [n], [L], 1.0)
    check(got, want, big, cache)
