"""Plans made on one stream and used on another, from the first operator that reads them on."""
import pytest
import torch

from tests.test_gpu_paged import F16, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("new,kv", [([1, 50], [3000, 700]), ([1, 1, 1], [40, 4000, 17])])
def test_append_and_attention_after_an_upload_that_waits(ops, new, kv):
    """The upload is queued behind work on its own stream; append and attention on the other one still see it."""
    H, Hk, D, page = 8, 2, 128, 16
    k, v, table = make_cache(kv, Hk, D, page, F16)
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(sum(new), (H + 2 * Hk) * D, generator=g).to(F16).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    k0, v0 = k.clone(), v.clone()
    q0 = ops.paged_append(qkv, k0, v0, table, plan.positions, plan.requests, H, rope_theta=1e4)
    want = ops.paged_attention(q0, k0, v0, table, plan)
    del plan
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(3):
        k1, v1 = k.clone(), v.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                big @ big
            late = ops.PagedPlan(new, kv, H, Hk, D, page)
        q = ops.paged_append(qkv, k1, v1, table, late.positions, late.requests, H, rope_theta=1e4)
        got = ops.paged_attention(q, k1, v1, table, late)
        del late
        torch.cuda.synchronize()
        assert torch.equal(q, q0) and torch.equal(k1, k0) and torch.equal(v1, v0) and torch.equal(got, want)
