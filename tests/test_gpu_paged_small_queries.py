"""bf16 queries of any size: an 8-bit cache's scales, or the caller's, bring their scores to ordinary ones.  A query
row is multiplied by a power of two on its way to f16, which is exact for bf16's 8 bits (but for values below 2^-39 of
the row's largest), so the bounds are those of ordinary queries."""
import pytest
import torch

from tests.paged8_bounds import Exact, check_rounding
from tests.paged8_util import BF16, E4M3, F16, I8, Cache
from tests.test_gpu_paged import check, make_cache, reference

pytestmark = pytest.mark.gpu

CALLS = [(4, 4, 128, [1, 1, 1], [1, 700, 5000]), (14, 2, 64, [1, 2, 1], [40, 333, 6000]), (8, 2, 128, [5, 17], [900, 300]),
         (8, 2, 64, [9, 30], [5000, 30]), (4, 2, 128, [257, 1, 64], [257, 2000, 4000]), (4, 4, 64, [300], [3000])]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def queries(rows, H, D, seed):
    g = torch.Generator().manual_seed(seed + 200)
    return (torch.randn(rows, H, D, generator=g) * 2).clamp(-7.9, 7.9).to(BF16).cuda()


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("power", [-118, -100, -40, -20, -10, -4, 16, 40, 100, 116])
@pytest.mark.parametrize("H,Hk,D,new,kv", CALLS)
def test_keys_of_the_other_size(ops, kind, power, H, Hk, D, new, kv):
    """Queries 2^power times as large against keys 2^-power times as large."""
    c = Cache(kv, Hk, D, 16, kind, seed=power + 200)
    c.ks *= 2.0 ** -power
    q = queries(sum(new), H, D, power) * 2.0 ** power
    assert torch.isfinite(q).all() and (c.ks[~torch.isnan(c.ks)] >= 2.0 ** -126).all()
    plan = ops.PagedPlan(new, kv, H, Hk, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, new, kv))


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("power", [-100, -40, -20])
@pytest.mark.parametrize("H,Hk,D,new,kv", CALLS)
def test_the_callers_scale(ops, kind, power, H, Hk, D, new, kv):
    """A scale that makes up for small queries: of all rows, and of every third one beside rows of large scores."""
    c = Cache(kv, Hk, D, 16, kind, seed=power + 200)
    q = queries(sum(new), H, D, power) * 2.0 ** power
    some = q.clone()
    some[::3, ::2] *= 2.0
    some[1::3, 1::2] = 0
    plan = ops.PagedPlan(new, kv, H, Hk, D, 16)
    for x in (q, some):
        scale = 2.0 ** -power * D ** -0.5
        got = ops.paged_attention(x, *c.args(), plan, scale=scale, **c.scales())
        assert ops.device_error() == 0
        check_rounding(got, Exact(c, x, new, kv, scale))


@pytest.mark.parametrize("power", [-120, -60, -20, -8])
@pytest.mark.parametrize("H,Hk,D,new,kv", CALLS)
def test_over_an_f16_cache(ops, power, H, Hk, D, new, kv):
    k, v, table = make_cache(kv, Hk, D, 16, F16, seed=power + 200, fill=float("nan"))
    q = queries(sum(new), H, D, power) * 2.0 ** power
    plan = ops.PagedPlan(new, kv, H, Hk, D, 16)
    scale = 2.0 ** -power * D ** -0.5
    got = ops.paged_attention(q, k, v, table, plan, scale=scale)
    assert ops.device_error() == 0
    want, big = reference(q, k, v, table, new, kv, scale)
    check(got, want, big, F16)


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_rows_of_every_size_in_one_call(ops, n):
    """Rows of 2^-60 .. 2^60 beside each other, rows of zeros, and rows whose own values differ by 2^30."""
    H, Hk, D, L = 8, 2, 128, 900
    c = Cache([L], Hk, D, 16, I8, seed=n)
    q = queries(n, H, D, n)
    power = torch.randint(-60, 6, (n, H, 1), generator=torch.Generator().manual_seed(n)).cuda()
    q = (q.float() * 2.0 ** power).to(BF16)
    q[:, 3] = 0
    q[:, 4, 1:] *= 2.0 ** -30
    q[:, 4, 0] = 4
    plan = ops.PagedPlan([n], [L], H, Hk, D, 16)
    got = ops.paged_attention(q, *c.args(), plan, **c.scales())
    assert ops.device_error() == 0
    check_rounding(got, Exact(c, q, [n], [L]))
