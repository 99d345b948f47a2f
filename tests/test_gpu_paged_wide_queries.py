"""bf16 queries past the range of an f16 cache's type: the scores are the formula's all the same.  The scale brings them
back to ordinary sizes, so the bounds are test_gpu_paged's own: a query value is rounded to f16's 11 bits after
division by a power of two, which is exact for bf16's 8."""
import pytest
import torch

from tests.test_gpu_paged import BF16, F16, check, make_cache, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("power", [15, 16, 17, 40, 100, 125])
@pytest.mark.parametrize("H,Hk,D,new,kv", [(4, 4, 128, [1, 1, 1], [1, 700, 5000]), (14, 2, 64, [1, 2, 1], [40, 333, 9000]),
                                           (8, 2, 128, [5, 17], [900, 300]), (8, 2, 64, [9, 30], [5000, 30]),
                                           (4, 2, 128, [257, 1, 64], [257, 2000, 4000]), (4, 4, 64, [300], [7000])])
def test_queries_beyond_the_caches_range(ops, power, H, Hk, D, new, kv):
    """All rows, and every third one beside rows of ordinary size (whose scores then are next to 0)."""
    page = 16
    k, v, table = make_cache(kv, Hk, D, page, F16, seed=power, fill=float("nan"))
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    g = torch.Generator().manual_seed(power)
    q = torch.randn(sum(new), H, D, generator=g).clamp(-3.9, 3.9).to(BF16).cuda()
    every = q * 2.0 ** power
    some = q.clone()
    some[::3, ::2] *= 2.0 ** power
    some[1::3, 1::2] *= 2.0 ** (power - 3)
    assert every.abs().max() > 65504 and torch.isfinite(every).all()
    for x in (every, some):
        scale = 2.0 ** -power * D ** -0.5
        got = ops.paged_attention(x, k, v, table, plan, scale=scale)
        assert ops.device_error() == 0
        want, big = reference(x, k, v, table, new, kv, scale)
        check(got, want, big, F16)


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_an_infinite_query_stays_in_its_row(ops, n):
    """NaN and infinite queries make their own (row, head) NaN and leave the others' bits."""
    H, Hk, D, L, page = 4, 2, 128, 700, 16
    k, v, table = make_cache([L], Hk, D, page, F16)
    plan = ops.PagedPlan([n], [L], H, Hk, D, page)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(n)).to(BF16).cuda()
    want = ops.paged_attention(q, k, v, table, plan)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[n // 2, 1, 9] = bad
        got = ops.paged_attention(x, k, v, table, plan)
        assert torch.isnan(got[n // 2, 1]).all()
        got[n // 2, 1] = want[n // 2, 1]
        assert torch.equal(got, want)
