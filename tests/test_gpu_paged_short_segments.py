"""Tensor-core attention over blocks of many short pieces of work: the two halves of a block hand over a barrier at
every tile that both meet, and neither may run a phase ahead, also where one is held up by its outputs."""
import pytest
import torch

from tests.test_gpu_paged import BF16, F16, check, make_cache, reference

pytestmark = pytest.mark.gpu

# Long requests beside ones of a tile or two; rows that see nothing; more items than blocks.
CASES = [
    ([230, 9, 10, 1, 18, 491, 101, 10, 46, 4, 31], [317, 148, 160, 99, 19, 5596, 100, 21, 44, 4, 81], 32, 8, 64, 256),
    ([591, 1, 7, 332, 225, 14], [4891, 165, 1, 325, 223, 11], 24, 8, 64, 32),
    ([1, 125, 7, 325, 4, 20, 201, 1], [3778, 115, 3, 2569, 0, 20, 201, 288], 51, 3, 128, 16),
    ([35, 0, 507], [30, 0, 4418], 80, 2, 128, 256),
    ([64] * 90, [64] * 90, 32, 8, 128, 16),
    ([40] * 120, [120] * 120, 16, 2, 64, 16),
    ([200, 200, 129, 130] * 12, [200, 700, 129, 90] * 12, 16, 16, 128, 64),
    ([33] * 60 + [300], [33] * 60 + [9000], 16, 2, 128, 16),
]


@pytest.mark.parametrize("types", [(F16, F16), (BF16, F16)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_blocks_of_many_short_pieces(case, types):
    from trifuse_b200 import ops
    new, kv, H, Hk, D, page = CASES[case]
    act, cache = types
    k, v, table = make_cache(kv, Hk, D, page, cache, seed=case, fill=float("nan"))
    q = (torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(case)) * 2).to(act).cuda()
    plan = ops.PagedPlan(new, kv, H, Hk, D, page)
    got = ops.paged_attention(q, k, v, table, plan)
    want, big = reference(q, k, v, table, new, kv)
    check(got, want, big, cache)
    out = torch.empty_like(got)
    for _ in range(40):
        for _ in range(10):
            ops.paged_attention(q, k, v, table, plan, out=out)
        assert ops.device_error() == 0, "a wait expired"
        assert torch.equal(out, got)
