"""Inputs and float64 restatements for the tests of the paged cache of 8 bits."""

import math

import torch

from tests.paged_helpers import EPS, make_table

BLOCK = 16


def scale_of(top: float) -> float:
    """The least power of two from 2^-126 on whose 127-fold reaches ``top``."""
    k = -126
    while 127.0 * math.ldexp(1.0, k) < top:
        k += 1
    return math.ldexp(1.0, k)


def fill(codes, scales, rows, slots, held):
    """Appends ``rows [tokens, Hkv, D]`` (float64) to codes and scales (host, changed
    in place); slots: (page, offset, position) of each, in order; held: positions
    that each token's sequence had before this step."""
    blocks = {}
    for t, (page, off, pos) in enumerate(slots):
        blocks.setdefault((page, off // BLOCK), []).append((t, off % BLOCK, pos))
    for (page, j), tokens in blocks.items():
        first = tokens[0][1]
        assert first == max(0, held[tokens[0][0]] - (tokens[0][2] - first))
        part = codes[page, :, j * BLOCK:(j + 1) * BLOCK]
        for h in range(codes.shape[1]):
            x = rows[[t for t, _, _ in tokens], h]
            old = float(scales[page, h, j]) if first else 0.0
            if not bool(torch.isfinite(x).all()) or math.isnan(old):
                scales[page, h, j] = float("nan")
                part[h, [o for _, o, _ in tokens]] = 0
                continue
            s = max(old, scale_of(float(x.abs().max())))
            if first and s != old:
                again = torch.round(part[h, :first].double() * (old / s))
                part[h, :first] = again.to(torch.int8)
            scales[page, h, j] = s
            part[h, [o for _, o, _ in tokens]] = torch.round(x / s).to(torch.int8)


def values(codes, scales):
    """What a pool holds, float64."""
    return (codes.double().view(*scales.shape, BLOCK, -1)
            * scales.double()[..., None, None]).view(codes.shape)


def empty_pool(pool, Hkv, page_size, D, seed):
    """Codes and scales of no sequence: any codes, scales that are not numbers."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-128, 128, (pool, Hkv, page_size, D), generator=g).to(torch.int8)
    return codes, torch.full((pool, Hkv, page_size // BLOCK), float("nan"))


def filled_pool8(table, pool, ctx, Hkv, D, page_size, seed, spread=0):
    """A pool whose blocks hold N(0,1) times a loudness of their own, of up to
    ``spread`` powers of two either way, where sequences lie; anything elsewhere."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = empty_pool(pool, Hkv, page_size, D, seed + 1)
    for s, c in enumerate(ctx):
        for b in range(-(-c // BLOCK)):
            page, j = int(table[s, b * BLOCK // page_size]), b * BLOCK % page_size // BLOCK
            n = min(BLOCK, c - b * BLOCK)
            loud = 2.0 ** ((2 * torch.rand(Hkv, generator=g) - 1) * (spread + 0.5))
            x = torch.randn(Hkv, n, D, generator=g) * loud[:, None, None]
            top = x.abs().amax((1, 2)).tolist()
            sc = torch.tensor([scale_of(t) for t in top])
            scales[page, :, j] = sc
            codes[page, :, j * BLOCK:j * BLOCK + n] = torch.round(
                x.double() / sc[:, None, None]).to(torch.int8)
    return codes, scales


def largest_weight(q, k, v_scales, table, ctx, new, page_size, scale):
    """The largest softmax weight times the largest value scale that each row sees,
    ``[T, Hq]`` (k: the keys' values)."""
    T, Hq, D = q.shape
    hg = Hq // k.shape[1]
    out, at = torch.zeros(T, Hq, dtype=torch.float64), 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        pos = torch.arange(c)
        page = table[s].long()[pos // page_size]
        for h in range(Hq):
            kk = k[page, h // hg, pos % page_size].double()
            vs = v_scales[page, h // hg, pos % page_size // BLOCK].double()
            for i in range(n):
                m = c - n + i + 1
                p = torch.softmax((kk[:m] @ q[at + i, h].double()) * scale, 0)
                out[at + i, h] = p.max() * vs[:m].max()
        at += n
    return out


def attention8_tolerance(ref, mag, size, largest, D, c, dtype):
    """Each element's bound: the output's rounding (half a step; fp16's numbers below
    2^-14 are 2^-24 apart, so 2^-25 there whatever their size); the weights' rounding for
    the second product, to fp16: half a step at most (2^-11, for fp32 two pieces, 2^-22),
    and 2^-25 where a row's largest weight (or weight times scale) is 2^12 or more: 2^-37
    of the largest for c codes of 127 times their scales at most; and fp32: a score is a sum of two products of pieces for
    each of D channels at most, pieces that leave 2^-22 of fp32 queries out, times a
    scale: off by (2 D + 10) 2^-24 of sum |q k| scale, which moves a weight and the
    weights' sum by that much relative each; exp2, the scales and the sums over c
    tokens add (3 c + 16) 2^-24 each."""
    eps, u = EPS[dtype], 2.0 ** -24
    moved = 2 * ((2 * D + 10) * u * size[..., None] + (3 * c + 16) * u)
    half = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    small = 127 * c * 2.0 ** -37 * largest[..., None]
    return (eps / 2) * ref.abs() + ((half + moved) * mag + small) * (1 + eps) + least


__all__ = ["BLOCK", "EPS", "make_table", "scale_of", "fill", "values", "empty_pool",
           "filled_pool8", "largest_weight", "attention8_tolerance"]
