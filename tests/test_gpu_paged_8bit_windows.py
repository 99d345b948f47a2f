"""Appends of many rows to an 8-bit cache with norms: windows of 16 rows, whose heads a block's warps share (more than 16
are read twice), an odd head at the end, against the formula in 64 bits."""
import pytest
import torch

from tests.paged8_util import BF16, E4M3, F16, I8, Cache
from tests.test_gpu_paged import append_reference, near
from tests.test_gpu_paged_8bit import append_check, clones

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("H,Hk,D", [(16, 16, 128), (4, 2, 64), (20, 5, 128), (17, 17, 64), (40, 40, 64), (3, 1, 128)])
@pytest.mark.parametrize("new", [[789], [700, 1, 130], [3] * 270, [17] * 50, [1] * 800])
def test_norms_over_windows(ops, act, kind, H, Hk, D, new):
    kv = [n + 5 + 3 * i % 40 for i, n in enumerate(new)]
    page = 32
    c = Cache(kv, Hk, D, page, kind)
    before = clones(c)
    g = torch.Generator().manual_seed(H)
    qkv = (torch.randn(sum(new), (H + 2 * Hk) * D, generator=g) * 1.5).to(act).cuda()
    qn, kn = ((1 + 0.2 * torch.randn(n * D, generator=g)).to(F16).cuda() for n in (H, Hk))
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    for theta in (1e4, None):
        q = ops.paged_append(qkv, *c.args(), plan.positions, plan.requests, H, q_norm=qn, k_norm=kn, rope_theta=theta,
                             **c.scales())
        wq, wk, wv = append_reference(qkv, H, Hk, D, plan.positions, qn, kn, 1e-5, theta)
        near(q, wq)
        append_check(c, before, (wk, wv), kv, [b - a for a, b in zip(new, kv)])
        for n, old in zip(("k", "v", "ks", "vs"), before):
            getattr(c, n).copy_(old)
