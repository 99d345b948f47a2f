"""Caches of 8-bit codes for the tests: made, read back and attended in 64 bits."""
import numpy as np
import torch

F16, BF16 = torch.float16, torch.bfloat16
I8, E4M3 = torch.int8, torch.float8_e4m3fn
LARGEST = {I8: 127.0, E4M3: 448.0}
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
BLOCK = 16


def encode(x, kind):
    """[..., page, D] -> codes, scales [..., page / 16]."""
    b = x.float().unflatten(-2, (-1, BLOCK))
    s = b.abs().amax((-1, -2)) / LARGEST[kind]
    y = b / torch.where(s > 0, s, 1.0)[..., None, None]
    y = y.round().to(I8) if kind == I8 else y.to(E4M3)
    return y.flatten(-3, -2), s


def decode(codes, scales):
    """float64 values."""
    return (codes.float().double().unflatten(-2, (-1, BLOCK)) * scales.double()[..., None, None]).flatten(-3, -2)


class Cache:
    """Shuffled pages of random tokens, whose blocks' magnitudes differ by up to 2^spread; past a length codes and
    scales hold anything (NaN codes of e4m3 and NaN scales among it)."""

    def __init__(self, lens, Hk, D, page, kind, seed=0, spread=3, spare=3):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
        self.lens, self.page, self.kind = lens, page, kind
        for n in "kv":
            x = torch.randn(pages, Hk, page, D, generator=g)
            x = x * 2.0 ** (spread * (torch.rand(pages, Hk, page // BLOCK, 1, 1, generator=g) - 0.5)).expand(
                -1, -1, -1, BLOCK, 1).reshape(pages, Hk, page, 1)
            codes, scales = encode(x, kind)
            setattr(self, n, codes)
            setattr(self, n + "s", scales)
        used = torch.zeros(pages, page, dtype=torch.bool)
        at = 0
        for r, n in enumerate(need):
            ids = order[at:at + n]
            self.table[r, :n] = ids
            used[ids.long()] = (torch.arange(n * page) < lens[r]).view(n, page)
            at += n
        stale = ~used
        for n in "kv":
            codes = getattr(self, n).view(torch.uint8)
            codes.transpose(1, 2)[stale] = 0x7f if kind == E4M3 else 0x81
            scales = getattr(self, n + "s")
            scales.transpose(1, 2)[stale.view(pages, -1, BLOCK).all(-1)] = float("nan")
        for n in ("k", "v", "ks", "vs", "table"):
            setattr(self, n, getattr(self, n).cuda())

    def args(self):
        return self.k, self.v, self.table

    def scales(self):
        return dict(k_scales=self.ks, v_scales=self.vs)

    def history(self, n, r, length):
        """[length, Hk, D] in float64 of "k" or "v"."""
        ids = self.table[r, : -(-length // self.page)].long()
        x = decode(getattr(self, n)[ids], getattr(self, n + "s")[ids]).transpose(1, 2)
        return x.reshape(-1, *x.shape[2:])[:length]


def attend(cache, q, new, kv, scale=None):
    """Outputs in 64 bits, and of each row the largest |v| it may see and the largest sum |q k| scale."""
    H, D = q.shape[1:]
    Hk = cache.k.shape[1]
    G = H // Hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    big = torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
    sums = torch.zeros_like(big)
    scale = D ** -0.5 if scale is None else scale
    row = 0
    for r, (n, L) in enumerate(zip(new, kv)):
        if n and L:
            k, v = cache.history("k", r, L), cache.history("v", r, L)
            qq = q[row:row + n].double().view(n, Hk, G, D)
            s = torch.einsum("nhgd,khd->nhgk", qq, k) * scale
            hidden = torch.arange(L, device=q.device)[None] > (L - n + torch.arange(n, device=q.device))[:, None]
            s = s.masked_fill(hidden[:, None, None], -np.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.where(s == -np.inf, 0.0, torch.exp(s - torch.where(m == -np.inf, 0.0, m)))
            l = e.sum(-1, keepdim=True)
            p = e / torch.where(l == 0, 1.0, l)
            # A key that the row does not see adds nothing, whatever its value.
            o = torch.einsum("nhgk,khd->nhgd", p, torch.nan_to_num(v))
            bad = torch.isnan(v).any(-1)  # [keys, heads]
            if bad.any():
                sees = ~hidden[:, None, :] & bad.T[None]
                o = o.masked_fill(sees.any(-1)[:, :, None, None], np.nan)
            out[row:row + n] = o.reshape(n, H, D)
            big[row:row + n] = torch.nan_to_num(v).abs().max()
            a = torch.einsum("nhgd,khd->nhgk", qq.abs(), torch.nan_to_num(k).abs()) * scale
            sums[row:row + n] = a.masked_fill(hidden[:, None, None], 0.0).amax((1, 2, 3))
        row += n
    return out, big, sums


def check(got, want, big, sums, rms=True):
    """Weights, f16 operands of the many-rows kernel and outputs are rounded once each.  A weight's (and a value's)
    rounding moves the output by 2^-11 max |v| at most; a key's by 2^-11 sum |q k| in the score, twice that in a
    weight relative to the others.  Over many roundings these average: each of the four adds 2^-11 / sqrt 3 of the
    output's norm, the keys' about twice that (scores of standard deviation two), so 2^-9 of the norm (f16) holds
    them with room, and 2^-8 for bf16 outputs (2^-8 / sqrt 3 of their own)."""
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    got, want = torch.where(fine, got, 0).double(), torch.where(fine, want, 0.0)
    assert torch.isfinite(got).all()
    u = UNIT[F16]
    weights = torch.expm1(4 * u * sums)[:, None, None]
    own = UNIT[BF16] * want.abs()
    err = (got - want).abs()
    bound = (2 * u + 1e-4 + weights) * big[:, None, None] + own + 1e-6
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.2f} of the bound"
    if rms and want.norm() > 0:
        limit = 2.0 ** -8
        assert (got - want).norm() <= limit * want.norm(), float((got - want).norm() / want.norm())
