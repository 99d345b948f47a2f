"""beam_select among many beams that lie closer than the rounding of their rows' sums: which of them are picked.

The beams of a request have the same logits, so their totals differ as their scores do, exactly; rows that begin at
different offsets from 16 bytes are summed in different orders."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def request(V, beams, steps, seed):
    g = torch.Generator().manual_seed(seed)
    row = torch.randn(1, 1, V, generator=g) * 2.5
    row[0, 0, V // 3] = 40.0  # nothing else comes near
    # steps of one unit in the last place of a number between 2 and 4
    order = torch.randperm(beams, generator=g) % steps
    scores = -(3.0 + order.float() * 2.0 ** -22)[None]
    return row.expand(1, beams, V).contiguous().cuda(), scores.cuda(), order


@pytest.mark.parametrize("V", [1001, 1003, 5003, 50303])
@pytest.mark.parametrize("beams,count,steps", [(8, 1, 1), (8, 3, 1), (64, 5, 1), (16, 4, 16), (64, 6, 64), (12, 2, 3)])
def test_more_beams_than_picked(ops, V, beams, count, steps):
    for seed in range(6):
        logits, scores, order = request(V, beams, steps, seed)
        got = ops.beam_select(logits, scores, count)
        want = torch.sort(order, stable=True).indices[:count]
        assert got.parent.cpu()[0].tolist() == want.tolist(), seed
        assert (got.token == V // 3).all()
    assert ops.device_error() == 0
