"""Arguments of the paged operators and of token_logprobs that need care at the entry: outputs and weights off their
alignment, integers of other types, caches of one head or one page."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged import BF16, F16, append_reference, check, make_cache, near, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("offset", [0, 1, 4, 8, 16])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_outputs_off_their_alignment(ops, offset, n):
    """out as a view that starts `offset` values into its storage: the same values, and nothing beside them."""
    H, Hk, D, page = 4, 2, 64, 16
    q, k, v, table, plan, want = run(ops, [n], [n + 5], H, Hk, D, page, F16, F16)
    wide = torch.full((n * H * D + 64,), 7.0, dtype=F16, device="cuda")
    out = wide[offset:offset + n * H * D].view(n, H, D)
    assert ops.paged_attention(q, k, v, table, plan, out=out) is out and torch.equal(out, want)
    assert (wide[:offset] == 7).all() and (wide[offset + n * H * D:] == 7).all()
    qkv = torch.randn(n, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(n)).to(F16).cuda()
    want = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H, rope_theta=1e4)
    wide.fill_(7.0)
    got = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H, rope_theta=1e4, out=out)
    assert got is out and torch.equal(out, want)
    assert (wide[:offset] == 7).all() and (wide[offset + n * H * D:] == 7).all()


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_norm_weights_off_their_alignment(ops, offset):
    """Both weights as slices of one buffer of parameters."""
    H, Hk, D, page, n = 4, 2, 64, 16, 5
    k, v, table = make_cache([n], Hk, D, page, F16)
    plan = ops.PagedPlan([n], [n], H, Hk, D, page)
    g = torch.Generator().manual_seed(offset)
    buffer = (1 + 0.2 * torch.randn(offset + (H + Hk) * D + 3, generator=g)).to(F16).cuda()
    qn, kn = buffer[offset:offset + H * D], buffer[offset + H * D + 3:offset + (H + Hk) * D + 3]
    qkv = torch.randn(n, (H + 2 * Hk) * D, generator=g).to(F16).cuda()
    q = ops.paged_append(qkv, k, v, table, plan.positions, plan.requests, H, q_norm=qn, k_norm=kn, rope_theta=1e4)
    wq, wk, _ = append_reference(qkv, H, Hk, D, plan.positions, qn, kn, 1e-5, 1e4)
    near(q, wq)
    near(k[table[0].long()].transpose(1, 2).reshape(-1, Hk, D)[:n], wk)


def test_top_of_any_integer_type(ops):
    x = torch.randn(3, 500, generator=torch.Generator().manual_seed(1)).cuda()
    t = torch.tensor([1, 2, 3], device="cuda")
    want = ops.token_logprobs(x, t, top=7)
    for top in (np.int64(7), np.int32(7), torch.tensor(7)):
        for a, b in zip(want, ops.token_logprobs(x, t, top=top)):
            assert torch.equal(a, b)
    for top in (7.0, np.float32(7), "7", None, np.int64(65)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, t, top=top)
