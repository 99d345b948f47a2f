"""token_logprobs where logits lie far out: masks by large finite values (down to the type's lowest), alone or beside
-inf, and rows whose own maximum is large.  Against the definition in 64 bits, under the bounds of
test_gpu_logprobs: differences of logits are exact or rounded once, whatever the logits' size."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import BF16, F16, F32, draw, reference, same

pytestmark = pytest.mark.gpu

LOWEST = {d: torch.finfo(d).min for d in (F32, F16, BF16)}
MASKS = [(F32, m) for m in (-1e5, -1e7, -1e9, -1e10, -1e20, -1e30, -1e32, -1e37, "lowest")] + [
    (BF16, m) for m in (-1e7, -1e10, -1e30, "lowest")] + [(F16, -3e4), (F16, "lowest")]


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def check(ops, logits, tokens, top):
    """The definition relative to each row's maximum (the same quotient; in 64 bits too, ln sum e^x loses its digits
    to a maximum of 1e20); order and ranks by the logits themselves."""
    r = ops.token_logprobs(logits, tokens, top=top)
    *_, rank, _, token = reference(logits, tokens, top)
    x = logits.double()
    far = x.amax(-1, keepdim=True)
    x = torch.where(torch.isfinite(far), x - far, x)
    lp, entropy, *_ = reference(x, tokens, top)
    top_lp = x.gather(1, token) - torch.logsumexp(x, -1, keepdim=True)
    same(r.logprob, lp, 1e-6, 4e-7)
    same(r.entropy, entropy, 1e-6 * (math.log(logits.shape[1]) + 1), 1e-6)
    assert torch.equal(r.rank.long(), rank) and torch.equal(r.top_token, token)
    same(r.top_logprob, top_lp, 1e-6, 4e-7)
    return r


@pytest.mark.parametrize("dtype,mask", MASKS)
@pytest.mark.parametrize("rows,V", [(10, 50304), (310, 9001), (160, 20483), (10, 40), (10, 250001)])
def test_masked_by_a_finite_value(ops, dtype, mask, rows, V):
    """Few tokens left, here and there, and none: rows on a cluster and on one block, full and partial tiles."""
    mask = LOWEST[dtype] if mask == "lowest" else mask
    x, t = draw(rows, V, dtype, seed=V)
    i = torch.arange(V, device="cuda")
    keep = [i == V - 1, i == 0, i == V // 2, i % 997 == 5, i < 3, i >= V - 20, i < V // 2, i >= 3 * V // 4, i < 0,
            i % 2 == 0]
    for r in range(rows):
        left = keep[r % 10]
        x[r] = torch.where(left, x[r], torch.full_like(x[r], mask))
        if r % 3 == 0 and left.any():
            t[r] = int(left.nonzero()[-1])
    for top in (0, 1, 20, 64):
        check(ops, x, t, min(top, V))
    x[:, ::3] = torch.where(x[:, ::3] == x.new_tensor(mask), -math.inf, x[:, ::3])
    check(ops, x, t, 5)


@pytest.mark.parametrize("dtype,at", [(F32, 2.0 ** 20), (F32, 1e6), (F32, 3e6), (F32, 1.5e9), (F32, 1e10), (F32, 1e30),
                                      (F32, 3e38), (BF16, 1e6), (BF16, 1e10), (BF16, 1e30), (BF16, 3e38), (F16, 6e4)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows,V", [(9, 50304), (300, 9001), (9, 40)])
def test_large_maxima(ops, dtype, at, sign, rows, V):
    """All logits near +-at: by the type's spacing there (ties and steps), by a few per cent, and beside small ones."""
    g = torch.Generator().manual_seed(V)
    centre = torch.tensor(sign * at, dtype=dtype).double()
    step = (torch.nextafter(centre.float(), torch.tensor(0.0)) - centre.float()).abs().double() if dtype == F32 else (
        centre.abs() * 2.0 ** (-8 if dtype == BF16 else -10))
    steps = torch.randint(0, 9, (rows, V), generator=g)
    near = centre - sign * steps * step
    wide = centre * (1 - 0.05 * torch.rand(rows, V, generator=g, dtype=torch.float64))
    few = torch.where(torch.rand(rows, V, generator=g) < 0.01, centre, torch.randn(rows, V, generator=g).double())
    t = torch.randint(0, V, (rows,), generator=g).cuda()
    for x in (near, wide, few):
        x = x.to(dtype).cuda()
        assert torch.isfinite(x).all()
        check(ops, x, t, 20)


def test_every_logit_the_lowest(ops):
    """Nothing but the type's lowest value: all tokens alike."""
    for dtype in (F32, F16, BF16):
        x = torch.full((3, 5000), LOWEST[dtype], dtype=dtype, device="cuda")
        r = check(ops, x, torch.tensor([0, 7, 4999], device="cuda"), 5)
        assert torch.allclose(r.logprob, torch.full_like(r.logprob, -math.log(5000)), atol=1e-5)
        assert r.rank.tolist() == [0, 7, 4999] and r.top_token[1].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("centre", [1e5, -1e6, 2e6, 5e6])
@pytest.mark.parametrize("rows,V", [(170, 57973), (230, 150001), (3, 250001)])
def test_long_rows_of_a_few_values(ops, centre, rows, V):
    """Logits a few steps of fp32 apart: hundreds of equal exponentials to a thread, whose sum may not drift."""
    g = torch.Generator(device="cuda").manual_seed(V)
    for std in (0.3, 2.5):
        x = torch.randn(rows, V, generator=g, device="cuda") * std + centre
        t = torch.randint(0, V, (rows,), generator=g, device="cuda")
        for top in (0, 8):
            check(ops, x, t, top)
