"""beam_select where totals reach the end of fp32: what is picked has a finite score, and the rest is none."""
import numpy as np
import pytest
import torch

from tests.test_gpu_beams import F16, F32, make

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def reference(logits, scores, count, finished=None, end=-1):
    """At 2^127 the steps of 64 bits swallow most logits, so equal totals are ordered by the beam, the logit, the token."""
    x, s = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    R, B, V = x.shape
    out = []
    for r in range(R):
        lists = []
        for b in range(B):
            if finished is not None and bool(finished[r, b]):
                lists.append([(s[r, b], b, 0.0, end)])
                continue
            m = x[r, b].max()
            if np.isfinite(m) and np.isfinite(s[r, b]):
                total = s[r, b] + (x[r, b] - m - np.log(np.exp(x[r, b] - m).sum()))
                lists.append(list(zip(total, [b] * V, x[r, b], range(V))))
        ranked = sorted((c for one in lists for c in one), key=lambda c: (-c[0], c[1], -c[2], c[3]))
        ranked = [c for c in ranked if np.isfinite(c[0])][:count]
        out.append(ranked + [(-np.inf, -1, 0.0, -1)] * (count - len(ranked)))
    best, parent, _, token = (torch.tensor([[c[i] for c in row] for row in out], dtype=torch.float64) for i in range(4))
    return best, parent.int(), token.long()


def check(ops, logits, scores, count, **kw):
    got = ops.beam_select(logits, scores, count, **kw)
    best, parent, token = reference(logits, scores, count, **kw)
    want = best.float()  # of falling totals: those beyond fp32 come last
    none = want == -torch.inf
    assert torch.equal(got.parent.cpu(), parent.masked_fill(none, -1))
    assert torch.equal(got.token.cpu(), token.masked_fill(none, -1))
    assert torch.equal(torch.isinf(got.score.cpu()), none)
    err = (got.score.double().cpu() - best).masked_fill(none, 0).abs()
    assert (err <= 5e-6 + 2.0 ** -24 * best.abs().masked_fill(none, 0)).all()
    assert ops.device_error() == 0
    return got


@pytest.mark.parametrize("V", [5, 1000, 20011])
@pytest.mark.parametrize("allowed", [1, 2, 7])
def test_masks_of_the_lowest_value(ops, V, allowed):
    """Fewer allowed tokens than are asked for, so masked ones go on; a step later their totals leave fp32."""
    B = 4
    logits, scores = make(3, B, V, F32, seed=V + allowed)
    logits[..., min(allowed, V):] = LOWEST
    scores[0, 1:] = -torch.inf
    scores[2] = -3.0e38
    first = check(ops, logits, scores, B)
    for count in (B, 12, 64):
        second = check(ops, logits, first.score, count)
    check(ops, logits, second.score[:, :B].contiguous(), B)


def test_scores_at_the_border(ops):
    """Totals on both sides of the last finite number, and on it."""
    scores = torch.tensor([[LOWEST, -3.0e38, -3.2e38, -2.0e38]], device="cuda")
    logits = torch.zeros(1, 4, 40, device="cuda")
    logits[..., 1:] = torch.linspace(-1e31, -3.4e38, 39, device="cuda")
    logits[0, 0, 1] = -2.0 ** 102
    logits[0, 0, 2] = -2.0 ** 103
    logits[0, 0, 3] = -2.0 ** 104
    for count in (1, 4, 64):
        check(ops, logits, scores, count)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_ended_beams_at_the_border(ops, dtype):
    logits, scores = make(2, 6, 300, dtype, seed=3)
    scores[:] = torch.tensor([LOWEST, -3.4e38, -3e38, -1e30, -5.0, -torch.inf])
    logits[..., 3:] = torch.finfo(dtype).min
    finished = torch.zeros(2, 6, dtype=torch.bool, device="cuda")
    finished[0, :3] = True
    check(ops, logits, scores, 20, finished=finished, end=9)
