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
