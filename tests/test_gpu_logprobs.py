"""token_logprobs against the definition in 64 bits.

The kernel sums fp32 exponentials (relative 2^-22 each) of exact differences;
log p = (x - m) - ln s carries a rounding of x - m (relative 2^-24), of ln s
and of the result, so 1e-6 absolute plus 4e-7 of its size covers it.  The
entropy subtracts two numbers of up to ln V + 1, each relative 1e-6.  Ranks,
alternatives and their order are exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def reference(logits, tokens, top):
    x = logits.double()
    V = x.shape[1]
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1)
    entropy = -torch.xlogy(p, p).sum(-1)
    given = (tokens >= 0) & (tokens < V)
    t = tokens.clamp(0, V - 1)
    xt = x.gather(1, t[:, None])
    lp = torch.where(given, xt[:, 0] - lse, math.nan)
    index = torch.arange(V, device=x.device)[None]
    rank = ((x > xt) | ((x == xt) & (index < t[:, None]))).sum(-1)
    fine = torch.isfinite(lse)
    rank = torch.where(given & fine, rank, -1)
    order = torch.nan_to_num(x, nan=-math.inf, posinf=math.inf, neginf=-1e300)
    token = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :top]
    nan = torch.full_like(lse, math.nan)
    return (torch.where(fine, lp, nan), torch.where(fine, entropy, nan), rank,
            torch.where(fine[:, None], x.gather(1, token) - lse[:, None], nan[:, None]), token)


def same(got, want, atol, rtol):
    assert got.dtype == F32
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    m = ~(torch.isnan(want) | inf)
    err = (got - want).abs()[m]
    assert (err <= atol + rtol * want.abs()[m]).all(), float(err.max())


def check(ops, logits, tokens, top):
    r = ops.token_logprobs(logits, tokens, top=top)
    lp, entropy, rank, top_lp, top_token = reference(logits, tokens, top)
    same(r.logprob, lp, 1e-6, 4e-7)
    same(r.entropy, entropy, 1e-6 * (math.log(logits.shape[1]) + 1), 1e-6)
    assert r.rank.dtype == torch.int32 and torch.equal(r.rank.long(), rank)
    assert torch.equal(r.top_token, top_token)
    same(r.top_logprob, top_lp, 1e-6, 4e-7)
    return r


def draw(rows, V, dtype, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * std).to(dtype).cuda()
    return x, torch.randint(0, V, (rows,), generator=g).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 65), (1, 4097), (5, 1000), (1, 50304), (64, 50304), (7, 32003),
                                    (300, 2049), (500, 151), (1, 250001)])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_shapes(ops, dtype, rows, V, top):
    x, t = draw(rows, V, dtype, seed=V)
    check(ops, x, t, min(top, V))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [9001, 9002, 9003, 9007])
def test_odd_strides(ops, dtype, V):
    """Rows that start at every offset from a 16-byte boundary."""
    x, t = draw(9, V + 11, dtype, seed=V)
    check(ops, x[:, 5:5 + V], (t % V), 7)
    check(ops, x.t().contiguous().t()[:, :V], t % V, 3)  # not contiguous at all


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("make", ["rising", "falling", "equal", "two values", "peaked", "signed zeros", "blocks"])
def test_orders(ops, dtype, make):
    """Values whose candidates overflow the buffer, ties, one certain token."""
    V, rows = 20011, 3
    i = torch.arange(V, dtype=F32)
    x = {"rising": i / 500, "falling": -i / 500, "equal": torch.full((V,), 1.5), "two values": (i % 7 == 3).float(),
         "peaked": torch.where(i == 777, 90.0, -30.0), "signed zeros": torch.where(i % 2 == 0, -0.0, 0.0),
         "blocks": torch.where((i // 4) % 256 < 224, 5.0 + (i % 97) / 97, -5.0)}[make]
    x = x.repeat(rows, 1).to(dtype).cuda()
    t = torch.tensor([0, 777, V - 1], device="cuda")
    for top in (1, 20, 64):
        check(ops, x, t, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("make", ["rising", "falling", "equal", "steps", "few threads", "late rise", "rising, with NaN"])
@pytest.mark.parametrize("rows", [20, 160])
def test_orders_of_long_rows(ops, dtype, make, rows):
    """Many candidates past the first tiles, where rows are shared by a cluster and where they are not."""
    V = 60001
    i = torch.arange(V, dtype=F32)
    noise = torch.randn(V, generator=torch.Generator().manual_seed(1))
    own = (i // (4 if dtype == F32 else 8)) % 128
    x = {"rising": i / 1000, "falling": -i / 1000, "equal": torch.zeros(V), "steps": (i // 9000) / 8,
         "few threads": torch.where((own > 2) & (own < 10), 10 + i / 4096, noise),
         "late rise": torch.where(i < 40000, noise, 5 + i / 8192),
         "rising, with NaN": torch.where(i % 6007 == 5, math.nan, i / 1000)}[make]
    x = x.repeat(rows, 1).to(dtype).cuda()
    t = (torch.arange(rows, device="cuda") * 977) % V
    for top in (1, 5, 20, 64):
        check(ops, x, t, top)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [40, 5000, 50304])
def test_infinities_and_nan(ops, dtype, V):
    x, t = draw(8, V, dtype, seed=3)
    x[0, 3] = -math.inf                 # one masked token, and it is asked for
    t[0] = 3
    x[1, :] = -math.inf                 # nothing left
    x[2, V // 2] = math.inf
    x[3, V - 1] = math.nan
    x[4, 1:] = -math.inf                # one certain token
    t[4] = 0
    x[5, : V - 2] = -math.inf           # fewer finite tokens than alternatives
    t[6], t[7] = -1, V                  # no token
    for top in (0, 5, 30):
        r = check(ops, x, t, top)
    assert r.logprob[4] == 0 and r.entropy[4] == 0 and r.logprob[0] == -math.inf
    assert r.rank[6] == -1 and torch.isnan(r.logprob[6]) and torch.isfinite(r.entropy[6])


def test_all_nan(ops):
    x = torch.full((2, 3000), math.nan, device="cuda")
    r = ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device="cuda"), top=5)
    assert torch.isnan(r.logprob).all() and torch.isnan(r.top_logprob).all()
    assert torch.equal(r.top_token, torch.arange(5, device="cuda").repeat(2, 1))


def test_leading_dimensions_and_far_values(ops):
    x, t = draw(12, 777, F32, std=300.0)
    a = ops.token_logprobs(x.view(3, 4, 777), t.view(3, 4), top=4)
    b = check(ops, x, t, 4)
    assert a.logprob.shape == (3, 4) and a.top_token.shape == (3, 4, 4)
    for u, v in zip(a, b):
        assert torch.equal(u.reshape(v.shape), v)
    one = ops.token_logprobs(x[0], t[0], top=2)
    assert one.logprob.shape == () and one.top_token.shape == (2,) and torch.equal(one.logprob, b.logprob[0])


def test_agrees_with_greedy(ops):
    x, t = draw(64, 50304, F32, seed=9)
    assert torch.equal(ops.token_logprobs(x, t, top=1).top_token[:, 0], ops.greedy_tokens(x))


def test_repeatable(ops):
    x, t = draw(3, 50304, F32, seed=4)
    a = ops.token_logprobs(x, t, top=20)
    for _ in range(20):
        for u, v in zip(a, ops.token_logprobs(x, t, top=20)):
            assert torch.equal(u, v)


def test_no_rows(ops):
    r = ops.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprob.shape == (0,) and r.top_token.shape == (0, 3)


def test_refusals(ops):
    x, t = draw(2, 100, F32)
    for a in ((x.double(), t, 0), (x, t[:1], 0), (x, t.int(), 0), (x, t, 65), (x, t, -1), (x[:, :10], t, 11),
              (x.cpu(), t, 0), (x, t.cpu(), 0), (x, t, 1.0)):
        with pytest.raises(ValueError):
            ops.token_logprobs(a[0], a[1], top=a[2])
