"""beam_select against its definition in 64 bits.

Scores are fp32 roundings of totals that are off by some 5e-6 at most (the sums of the rows); what is picked has to be
what 64 bits pick, ties by the lower beam, then the lower token."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def reference(logits, scores, count, finished=None, end=-1):
    x, s = logits.double().cpu(), scores.double().cpu()
    R, B, V = x.shape
    m = x.amax(-1, keepdim=True)
    ok = torch.isfinite(m[..., 0]) & torch.isfinite(s)
    total = s[..., None] + (x - m - torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    total[~ok] = -np.inf
    token = torch.arange(V).expand(R, B, V).clone()
    if finished is not None:
        f = finished.cpu()
        total[f] = -np.inf
        total[..., 0][f] = torch.where(torch.isfinite(s[f]), s[f], -np.inf)
        token[..., 0][f] = end
    best, at = torch.sort(total.view(R, -1), dim=-1, descending=True, stable=True)
    if best.shape[1] < count:
        pad = count - best.shape[1]
        best, at = torch.nn.functional.pad(best, (0, pad), value=-np.inf), torch.nn.functional.pad(at, (0, pad))
    best, at = best[:, :count], at[:, :count]
    none = best == -np.inf
    return best, torch.where(none, -1, at // V).int(), torch.where(none, -1, token.view(R, -1).gather(1, at))


def check(ops, logits, scores, count=None, **kw):
    got = ops.beam_select(logits, scores, count, **kw)
    count = logits.shape[1] if count is None else count
    best, parent, token = reference(logits, scores, count, **kw)
    assert got.score.shape == got.parent.shape == got.token.shape == (logits.shape[0], count)
    assert (got.score.dtype, got.parent.dtype, got.token.dtype) == (torch.float32, torch.int32, torch.int64)
    assert torch.equal(got.parent.cpu(), parent) and torch.equal(got.token.cpu(), token)
    g = got.score.double().cpu()
    assert torch.equal(torch.isinf(g), torch.isinf(best))
    err = torch.where(torch.isinf(best), 0, g - best)
    assert (err.abs() <= 5e-6 + 2.0 ** -24 * best.abs().nan_to_num(posinf=0, neginf=0)).all(), float(err.abs().max())
    assert ops.device_error() == 0
    return got


def make(R, B, V, dtype=F32, seed=0, std=2.5, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(R, B, V, generator=g) * std).to(dtype).cuda(),
            (torch.randn(R, 1, generator=g) * 20 - 60 + torch.randn(R, B, generator=g) * spread).cuda())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("R,B,V,count", [(1, 1, 50304, 1), (1, 4, 50304, 4), (3, 5, 1000, 10), (64, 8, 5003, 8), (2, 64, 777, 64),
                                         (300, 3, 130, 6), (40, 16, 20011, 32), (1, 2, 152000, 64)])
def test_shapes(ops, dtype, R, B, V, count):
    check(ops, *make(R, B, V, dtype, seed=V), count)


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 31, 63, 64, 65, 255])
@pytest.mark.parametrize("count", [1, 5, 64])
def test_small_vocabularies(ops, V, count):
    """Fewer continuations than asked for: the rest is none."""
    for B in (1, 3):
        check(ops, *make(2, B, V, F32, seed=V), count)


def test_flat_and_tied(ops):
    """Equal logits, equal beams, both: ties go to the lower beam, then the lower token."""
    logits, scores = make(3, 4, 5000)
    logits[0] = 1.25
    scores[0] = -3.0
    logits[1] = logits[1, :1]
    scores[1] = -7.5
    logits[2] = logits[2].round()
    check(ops, logits, scores, 16)
    check(ops, logits.bfloat16(), scores, 16)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_near_totals_are_told_apart(ops, dtype):
    """Beams whose best totals lie a few 1e-9 apart, far below the passes' rounding: the order is that of 64 bits."""
    R, B, V = 32, 6, 3000
    logits, _ = make(R, B, V, dtype, seed=3)
    x = logits.double()
    top = torch.log_softmax(x, -1).amax(-1)
    target = -20.0
    # fp32 scores that bring every beam's best continuation as close to the target as they can
    scores = (target - top).float()
    gaps = (scores.double() + top).sort(-1).values.diff(dim=-1)
    assert (gaps.abs() < 2e-6).all() and (gaps.abs() > 0).any()
    check(ops, logits, scores, B)


def test_finished_beams(ops):
    logits, scores = make(20, 6, 4000, seed=5, spread=4)
    g = torch.Generator().manual_seed(9)
    finished = (torch.rand(20, 6, generator=g) < 0.4).cuda()
    finished[0] = True
    finished[1] = False
    logits[finished] = float("nan")  # not read
    check(ops, logits, scores, 6, finished=finished, end=17)
    check(ops, logits, scores, 12, finished=finished, end=-5)


def test_beams_that_are_none(ops):
    """Scores of -inf (the first step's other beams), NaN and +inf; rows of NaN, +inf and -inf; nothing left at all."""
    nan, inf = float("nan"), float("inf")
    logits, scores = make(9, 4, 3000, seed=6)
    scores[0, 1:] = -inf
    scores[1, 0], scores[1, 2] = nan, inf
    logits[2, 1, 77] = nan
    logits[3, 0, 78] = inf
    logits[4, 3] = -inf
    logits[5, :, 10:] = -inf
    logits[6, :, 1:] = -inf
    scores[7] = -inf
    logits[8, :] = -inf
    check(ops, logits, scores, 4)
    check(ops, logits, scores, 50)


def test_masks_and_far_logits(ops):
    """Masks of the type's lowest value, -inf and -1e30; rows that lie far out as a whole."""
    logits, scores = make(6, 4, 9000, seed=7)
    logits[0, :, ::2] = torch.finfo(F32).min
    logits[1, :, 5:] = -float("inf")
    logits[2, :, 3:] = -1e30
    logits[3] = logits[3] - 5e6
    logits[4] = logits[4] * 100 + 3e6
    logits[5, 1] = -1e30
    check(ops, logits, scores, 4)


@pytest.mark.parametrize("order", ["rising", "falling", "equal ends"])
def test_order_of_the_row(ops, order):
    logits, scores = make(2, 3, 20000, seed=8)
    if order == "equal ends":
        logits[..., :5000] = logits[..., -5000:] = 9.0
    else:
        logits = logits.sort(-1, descending=order == "falling").values
    check(ops, logits, scores, 40)


def test_strides(ops):
    """Rows apart, a slice of a wider buffer, requests that are not evenly apart, transposed, expanded; a row that
    starts off 16 bytes."""
    logits, scores = make(3, 4, 1001, seed=2)
    want = check(ops, logits, scores)
    wide = torch.full((3, 4, 1300), 1e9, device="cuda")
    wide[..., 7:1008] = logits
    apart = torch.full((3, 6, 1001), 1e9, device="cuda")
    apart[:, :4] = logits
    for view in (wide[..., 7:1008], apart[:, :4], logits.transpose(0, 1).contiguous().transpose(0, 1),
                 logits.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = ops.beam_select(view, scores.t().contiguous().t())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(ops, logits[:, :1].expand(3, 4, 1001), scores)
    check(ops, logits[:1].expand(3, 4, 1001), scores)


def test_repeatable_streams_and_capture(ops):
    logits, scores = make(16, 8, 50304, seed=4)
    want = check(ops, logits, scores)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(ops.beam_select(logits, scores), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(logits, scores)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.beam_select(logits, scores)
    other, _ = make(16, 8, 50304, seed=40)
    for x in (logits.clone(), other):
        logits.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        again = ops.beam_select(logits, scores)
        assert all(torch.equal(a, b) for a, b in zip(held, again))


def test_no_requests(ops):
    got = ops.beam_select(torch.empty(0, 4, 100, device="cuda"), torch.empty(0, 4, device="cuda"))
    assert got.score.shape == (0, 4)


def test_refusals(ops):
    from trifuse_b200 import TriFuseError
    logits, scores = make(2, 3, 100)
    finished = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for args, kw in (((logits.int(), scores), {}), ((logits[0], scores), {}), ((logits, scores[:1]), {}),
                     ((logits, scores.double()), {}), ((logits, scores, 0), {}), ((logits, scores, 65), {}),
                     ((logits, scores), dict(finished=finished.int())), ((logits, scores), dict(finished=finished[:1])),
                     ((logits.cpu(), scores), {}), ((logits, scores.cpu()), {}), ((logits[..., :0], scores), {})):
        with pytest.raises((ValueError, TriFuseError)):
            ops.beam_select(*args, **kw)
    with pytest.raises((ValueError, TriFuseError)):
        ops.beam_select(torch.zeros(1, 65, 8, device="cuda"), torch.zeros(1, 65, device="cuda"))
    for kw in (dict(count=1.5), dict(end=1.5)):
        with pytest.raises(TypeError):
            ops.beam_select(logits, scores, **kw)
