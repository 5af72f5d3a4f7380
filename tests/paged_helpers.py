"""Inputs and float64 restatements for the tests of the paged cache."""

import numpy as np
import torch

EPS = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}


def make_table(lens, page_size, seed, spare=5):
    """Scattered pages for sequences of ``(before, new)`` tokens: the table, the
    pool's size, context lengths and new lengths.  Entries behind a sequence's
    last page are invalid on purpose."""
    ctx = [b + n for b, n in lens]
    pages = [-(-c // page_size) for c in ctx]
    pool = sum(pages) + spare
    order = np.random.RandomState(seed).permutation(pool)
    table = np.full((len(lens), max(pages + [1]) + 1), -1, dtype=np.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    return torch.from_numpy(table), pool, ctx, [n for _, n in lens]


def slots_of(table, ctx, new, page_size):
    """(page, offset, position) of each new token, in the plan's order."""
    out = []
    for s, (c, n) in enumerate(zip(ctx, new)):
        for p in range(c - n, c):
            out.append((int(table[s, p // page_size]), p % page_size, p))
    return out


def filled_pool(table, pool, ctx, Hkv, D, page_size, dtype, seed):
    """K and V pages (host): N(0,1) where sequences lie, NaN everywhere else."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.full((pool, Hkv, page_size, D), float("nan"), dtype=dtype)
        for s, c in enumerate(ctx):
            for j in range(-(-c // page_size)):
                m = min(page_size, c - j * page_size)
                x[int(table[s, j]), :, :m] = torch.randn(Hkv, m, D, generator=g).to(dtype)
        out.append(x)
    return out


def sequence_kv(pages, table, s, c, page_size):
    """``[Hkv, c, D]`` of sequence s, in the pages' type."""
    idx = table[s, :-(-c // page_size)].long()
    x = pages[idx].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :c]


def attention64(q, k_pages, v_pages, table, ctx, new, page_size, scale):
    """The formula in float64 on the host, with what the tolerances need: outputs,
    sum p |v| and the largest sum |q k| * scale of each row."""
    T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    hg = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    mag, size = torch.zeros_like(out), torch.zeros(T, Hq, dtype=torch.float64)
    at = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        k = sequence_kv(k_pages, table, s, c, page_size).double()
        v = sequence_kv(v_pages, table, s, c, page_size).double()
        for h in range(Hq):
            kv = h // hg
            qq = q[at:at + n, h].double()
            for i in range(n):
                m = c - n + i + 1
                z = (k[kv, :m] @ qq[i]) * scale
                p = torch.softmax(z, 0)
                out[at + i, h] = p @ v[kv, :m]
                mag[at + i, h] = p @ v[kv, :m].abs()
                size[at + i, h] = (k[kv, :m].abs() @ qq[i].abs()).max() * scale
        at += n
    return out, mag, size


def attention_tolerance(ref, mag, size, D, c, dtype):
    """Each element's bound: the output's rounding (half a step); the weights'
    rounding to a 16-bit type (half a step of each p |v|; their sum is not
    rounded); and fp32: a score is a sum of D products, off by at most
    (D + 3) 2^-24 of sum |q k| scale (D sums, the scale, its own rounding and the
    reference's maximum), which moves a weight and the weights' sum by that
    much relative each; exp2 and the sums over c tokens add (c + 8) 2^-24 each."""
    eps = EPS[dtype]
    u = 2.0 ** -24
    moved = 2 * ((D + 3) * u * size[..., None] + (c + 8) * u)
    half = eps / 2 if dtype != torch.float32 else 0.0
    return (eps / 2) * ref.abs() + (half + moved) * mag * (1 + eps) + 1e-30


def rows64(x, w, cos, sin, interleaved, eps=1e-6):
    """Norm and rotation of ``[T, H, D]`` rows in float64 (cos, sin ``[T, r/2]``)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    if cos is None:
        return y
    r = 2 * cos.shape[-1]
    i = torch.arange(r // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    out = y.clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out
