"""A key that outweighs all others over a long history: the others' weights are tiny one by one, and count together.
An output stays within test_gpu_paged's bound (the weights' relative rounding times the largest value, the output's
own, fp32 noise), so weights may not vanish in the cache's 16-bit type."""
import math

import pytest
import torch

from tests.test_gpu_paged import BF16, F16, UNIT, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("gap", [9.0, 12.0, 15.0, 17.0, 17.47, 18.5, 20.0])
@pytest.mark.parametrize("B,n,G,L,D,sinks", [
    (1, 200, 1, 60000, 64, [0]), (1, 20, 2, 60000, 128, [0]), (3, 300, 1, 40000, 128, [0, 7]),
    (148, 200, 1, 60000, 64, [0]), (296, 40, 1, 60000, 64, [0]),
    (1, 1, 1, 60000, 64, [0]), (148, 1, 1, 400000, 64, [0, 32, 64, 96]), (148, 4, 4, 400000, 64, [0, 32, 64, 96])])
def test_many_small_weights_count(ops, act, cache, gap, B, n, G, L, D, sinks):
    """Scores 0 but for the sinks' gap; values 0 at the sinks, about 1 elsewhere: an output is the others' share."""
    page = 256
    pages = -(-L // page)
    k = torch.zeros(pages, 1, page, D, dtype=cache, device="cuda")
    v = torch.ones_like(k)
    v[..., 1::2] = 0.75
    for s in sinks:
        k[s // page, 0, s % page, 0] = gap
        v[s // page, 0, s % page] = 0
    gap = float(k[0, 0, sinks[0], 0])  # as the type holds it
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].repeat(B, 1)  # the requests share their pages
    q = torch.zeros(B * n, G, D, dtype=act, device="cuda")
    q[..., 0] = 1
    plan = ops.PagedPlan([n] * B, [L] * B, G, 1, D, page)
    got = ops.paged_attention(q, k, v, table, plan, scale=1.0).double()
    assert ops.device_error() == 0
    others = torch.arange(L - n + 1, L + 1, dtype=torch.float64, device="cuda") - len(sinks)
    mass = others * math.exp(-gap)
    want = (mass / (mass + len(sinks))).repeat(B)[:, None, None] * v[-1, 0, 0].double()
    err = (got - want).abs()
    bound = UNIT[cache] + UNIT[act] * want + 1e-4 + 1e-6
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("act,cache", TYPES)
def test_large_values_do_not_overflow(ops, act, cache, n):
    """Values at f16's end (and far up in bf16) with every weight alike: the average, no infinity on the way."""
    L, D, page = 3000, 64, 16
    top = 65504.0 if cache == F16 else 1e34
    k = torch.zeros(-(-L // page), 2, page, D, dtype=cache, device="cuda")
    v = torch.full_like(k, top)
    table = torch.arange(len(k), dtype=torch.int32, device="cuda")[None]
    q = torch.ones(n, 4, D, dtype=act, device="cuda")
    plan = ops.PagedPlan([n], [L], 4, 2, D, page)
    got = ops.paged_attention(q, k, v, table, plan).double()
    want = float(v[0, 0, 0, 0].double())
    want = float(torch.tensor(want).to(act).double()) if act == BF16 else want
    assert ((got - want).abs() <= 2 * UNIT[act] * want).all()
