"""What 8-bit paged attention may be off by, from what it rounds: each weight once, to f16, and the output, to its own
type.  Codes are exact in f16, scales and scores are fp32."""
import torch

from tests.paged8_util import F16, LARGEST, UNIT

LEAST = {F16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step below the type's normal numbers


class Exact:
    """One call in 64 bits: want [rows, H, D]; of each output sum p |v| (mass), sum (p v)^2 (squares) and its largest
    term; of each row and head a score's largest sum |q k| scale (sums), and the largest p s_v (share) by the keys."""

    def __init__(self, cache, q, new, kv, scale=None):
        H, D = q.shape[1:]
        Hk = cache.k.shape[1]
        G = H // Hk
        scale = D ** -0.5 if scale is None else scale
        f64 = dict(dtype=torch.float64, device=q.device)
        self.want, self.mass, self.squares, self.top = (torch.zeros(q.shape, **f64) for _ in range(4))
        self.sums, self.share = (torch.zeros(q.shape[:2] + (1,), **f64) for _ in range(2))
        row = 0
        for r, (n, L) in enumerate(zip(new, kv)):
            if n and L:
                k, v = cache.history("k", r, L), cache.history("v", r, L)  # [L, Hk, D]
                ids = cache.table[r, : -(-L // cache.page)].long()
                unit = cache.vs[ids].double().permute(0, 2, 1).reshape(-1, Hk).repeat_interleave(16, 0)[:L]
                keys = torch.arange(L, device=q.device)[None]
                hidden = (keys > (L - n + torch.arange(n, device=q.device))[:, None])[:, None, None]
                at = slice(row, row + n)
                qq = q[at].double().view(n, Hk, G, D)
                s = (torch.einsum("nhgd,khd->nhgk", qq, k) * scale).masked_fill(hidden, -torch.inf)
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - torch.where(m == -torch.inf, 0.0, m))
                l = e.sum(-1, keepdim=True)
                p = e / torch.where(l == 0, 1.0, l)

                def outputs(x, y):
                    return torch.einsum("nhgk,khd->nhgd", x, y).reshape(n, H, D)

                self.want[at] = outputs(p, v)
                self.mass[at] = outputs(p, v.abs())
                self.squares[at] = outputs(p * p, v * v)
                shares = p * unit.T[None, :, None]
                most, which = shares.max(-1)  # [n, Hk, G]
                heads = torch.arange(Hk, device=q.device)[None, :, None].expand_as(which)
                self.top[at] = (p.gather(-1, which[..., None]) * v[which, heads]).reshape(n, H, D).square()
                self.share[at] = (most * LARGEST[cache.kind] * L).reshape(n, H, 1)
                a = torch.einsum("nhgd,khd->nhgk", qq.abs(), k.abs()) * scale
                self.sums[at] = a.masked_fill(hidden, 0.0).amax(-1).reshape(n, H, 1)
            row += n

    def rows(self, at):
        """The same of some rows."""
        some = object.__new__(Exact)
        some.__dict__.update({n: x[at] for n, x in self.__dict__.items()})
        return some


def check_rounding(got, ref, scattered=True, largest_exact=False, exponents=2.0 ** -18):
    """Each output: 2^-11 of sum p |v| for the weights (2^-32 of the largest share for each that lies below f16's
    normal numbers), its own rounding, and fp32's part: eight sums' roundings (2^-23) of a score's terms and the
    exponents' own (the scales' logarithms, up to 2^6, are within 2^-19; up to 2^9, added up in three steps, 2^-13 for
    the calls that say so), in numerator and denominator.

    All outputs together, where values and shares are scattered: independent roundings add up by their squares.  A
    relative error evenly spread up to u has u^2 / 3 times the mean of 1 / m^2 over mantissas, 0.541 where they are
    spread over their logarithm: 0.18 u^2 for each term p v.  The outputs' own is taken from their 64-bit values; 15 per
    cent of room.  largest_exact: the largest share counts as not rounded."""
    act, want = got.dtype, ref.want
    assert torch.isfinite(want).all() and torch.isfinite(got).all()
    u, own = UNIT[F16], UNIT[act]
    err = (got.double() - want).abs()
    fp32 = 2 * (exponents + 16 * 2.0 ** -23 * ref.sums) * ref.mass
    bound = u * ref.mass + 2.0 ** -32 * ref.share + fp32 + own * (want.abs() + u * ref.mass + fp32) + LEAST[act]
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.2f} of the bound"
    if scattered:
        rounded = (want.to(act).double() - want).square().sum()
        squares = ref.squares - ref.top if largest_exact else ref.squares
        limit = 1.15 * (rounded + 0.18 * u * u * squares.clamp_min(0).sum() + fp32.square().sum()).sqrt()
        total = err.square().sum().sqrt()
        assert total <= limit, f"{float(total / rounded.sqrt()):.2f} times the outputs' own rounding, {float(limit / rounded.sqrt()):.2f} allowed"
