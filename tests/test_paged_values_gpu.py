"""GPU tests of the paged cache's special values: infinities and NaN that a token
sees, weights far below a row's largest, the bits of a copy."""

import pytest
import torch

from tests.paged_helpers import EPS, attention64, attention_tolerance
from tests.test_paged_gpu import _attend, _c, _setup

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _slot(pages, table, s, pos, page_size):
    """The pool's ``[Hkv, D]`` of a sequence's position."""
    return pages[int(table[s, pos // page_size]), :, pos % page_size]


def _same(o, ref, tol):
    """Finite elements within the bound, the others the same."""
    o = o.double().cpu()
    fine = torch.isfinite(ref)
    assert bool(((o - ref).abs() <= tol)[fine].all())
    assert torch.equal(torch.isnan(o), torch.isnan(ref))
    big = torch.isinf(ref)
    assert torch.equal(o[big], ref[big])
    return fine


@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_infinities_that_all_rows_see(hip_device, dtype, D, n):
    """Wherever the position lies: in a step of positions that every row sees to its
    end, in one that some do not, in a split of the context."""
    case = _setup([(70, n), (1500, n), (9, 1)], 16, dtype, 4, 2, D, seed=9)
    table, pool, ctx, new, kp, vp, plan, q = case
    for s, positions in ((0, (0, 13, 40, 69)), (1, (3, 64, 700, 1499)), (2, (4,))):
        for i, pos in enumerate(positions):
            v = _slot(vp, table, s, pos, 16)
            v[0, 7 * i] = INF
            v[1, 7 * i + 1] = -INF
            v[1, 7 * i + 2] = NAN
            v[:, 60] = INF if i % 2 == 0 else -INF          # (both: NaN)
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 16, D ** -0.5)
    fine = _same(_attend(case), ref, attention_tolerance(ref, mag, size, D, max(ctx), dtype))
    assert not fine[0, :, 60].any() and fine[:, :, 61].all()


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 24])
def test_an_infinity_of_little_weight(hip_device, dtype, n):
    """Every weight is positive: e^-40 of the largest too."""
    D = 64
    case = _setup([(300, n)], 32, dtype, 2, 2, D, seed=4)
    table, pool, ctx, new, kp, vp, plan, q = case
    q[:] = 1.0
    for pos in (5, 100):
        _slot(kp, table, 0, pos, 32)[:] = -5.0              # score -40, the others' N(0,1)
        _slot(vp, table, 0, pos, 32)[:, 3] = INF
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 32, D ** -0.5)
    assert bool((ref[:, :, 3] == INF).all())
    _same(_attend(case), ref, attention_tolerance(ref, mag, size, D, max(ctx), dtype))


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 24])
def test_an_infinity_in_a_split_of_no_weight(hip_device, dtype, n):
    """A split of the context whose scores all lie 140 nats below another's (2^-202:
    nothing in fp32), with an infinity in it."""
    D = 64
    case = _setup([(3000, n)], 32, dtype, 2, 2, D, seed=4)
    table, pool, ctx, new, kp, vp, plan, q = case
    assert list(plan._info)[5] > 0
    q[:] = 1.0
    for pos in range(1500):
        _slot(kp, table, 0, pos, 32)[:] = -17.5
    _slot(vp, table, 0, 3, 32)[:, 3] = INF
    _slot(vp, table, 0, 3, 32)[1, 4] = -INF
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 32, D ** -0.5)
    assert bool((ref[:, :, 3] == INF).all()) and bool((ref[:, 1, 4] == -INF).all())
    _same(_attend(case), ref, attention_tolerance(ref, mag, size, D, max(ctx), dtype))


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_keys_that_are_not_finite_leave_no_finite_row(hip_device, dtype):
    """A NaN score: the whole row is NaN, as the formula has it, and no other."""
    for n in (1, 24):
        case = _setup([(300, n), (50, 1)], 32, dtype, 4, 2, 64, seed=4)
        table, pool, ctx, new, kp, vp, plan, q = case
        _slot(kp, table, 0, 17, 32)[1, 3] = NAN
        o = _attend(case).cpu()
        assert bool(torch.isnan(o[:n, 2:]).all())
        assert bool(torch.isfinite(o[:n, :2]).all()) and bool(torch.isfinite(o[n:]).all())


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("below,spread", [(25.2, 0.0), (22.0, 0.0), (21.0, 0.3), (12.0, 1.0)])
def test_a_long_tail_below_the_largest(hip_device, dtype, n, below, spread):
    """16K positions, every 32nd of them ``below`` log2 units above the others, whose
    values alone count.

    The bound: the output's rounding; the weights' (half a step of a 16-bit type; an
    fp16 weight is held as 2^7 of the largest at least, so half a step of its smallest
    numbers is 2^-32 of the largest weight, of which the sum has c / 32 - 1 or more);
    and fp32's.  Of these a score is a sum of D products, off by (D + 3) 2^-24 of
    sum |q k| scale, which moves a weight and the weights' sum by that each; a lane adds
    at most half of the positions one after the other, each off by 2^-24 of the sum, for
    the weights and (in matrix products of 16 positions) for the values."""
    D, c, hg, much = 64, 16384, 4, 1000.0
    case = _setup([(c - n, n)], 64, dtype, hg, 1, D, seed=7)
    table, pool, ctx, new, kp, vp, plan, q = case
    g = torch.Generator().manual_seed(3)
    q[:] = 1.0
    k, v = torch.zeros(c, D), torch.full((c, D), much)
    k[:, :16] = spread * torch.randn(c, 16, generator=g)
    k[::32] = below * 0.6931471805599453 / 8.0              # (64 channels, the scale is 1/8)
    v[::32] = 0.0
    for j in range(c // 64):
        kp[int(table[0, j]), 0], vp[int(table[0, j]), 0] = (
            x[64 * j:64 * j + 64].to(dtype) for x in (k, v))
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 64, D ** -0.5)
    u, half = 2.0 ** -24, EPS[dtype] / 2
    fp32 = 2 * ((D + 3) * u * size[..., None] + (c / 2 + 64) * u)
    tol = half * ref.abs() + ((half if dtype != FF else 0.0) + fp32) * mag * (1 + 2 * half)
    if dtype == HF:
        tol = tol + c * much * 2.0 ** -32 / (c / 32 - 1)
    err = (_attend(case).double().cpu() - ref).abs()
    print(f"[tail] {dtype} n={n} {below} worst {float((err / tol).max()):.3f} of the bound")
    assert bool((err <= tol).all())


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_single_tokens_are_as_exact_beside_many_rows(hip_device, dtype, D):
    """Their weights enter the second product in two pieces (off by 2^-18 at most:
    half a step of half a step), alone or in the launch of a sequence of many rows."""
    lens, Hq, Hkv = [(60, 1), (100, 40), (90, 1), (33, 3)], 8, 2
    case = _setup(lens, 16, dtype, Hq, Hkv, D, seed=5)
    table, pool, ctx, new, kp, vp, plan, q = case
    q *= 0.2
    assert list(plan._info)[6:9] == [0, 0, 0]               # (one launch)
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 16, D ** -0.5)
    u = 2.0 ** -24
    moved = 2 * ((D + 3) * u * size[..., None] + (max(ctx) + 8) * u)
    tol = EPS[dtype] / 2 * ref.abs() + (2.0 ** -18 + moved) * mag * (1 + EPS[dtype])
    if dtype == HF:
        tol = tol + max(ctx) * mag * 2.0 ** -32
    err = (_attend(case).double().cpu() - ref).abs()
    rows = [0] + list(range(41, 45))
    print(f"[company] {dtype} D={D} worst {float((err / tol)[rows].max()):.3f} of the bound")
    assert bool((err <= tol)[rows].all())


# ------------------------------------------------------- the append's copies
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rotary", [0, 32])
def test_every_bit_of_a_copy(hip_device, dtype, offset, rotary):
    """All 65536 patterns, signalling NaN among them: values, and channels that are
    neither normed nor rotated, from rows on and off 16-byte borders."""
    T, H, D, page = 512, 2, 64, 32
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    flat = torch.empty(65536 + offset, dtype=torch.int16, device="cuda:0")
    flat[offset:] = bits.cuda()
    x = flat[offset:].view(dtype).view(T, H, D)
    table = torch.randperm(T // page, generator=torch.Generator().manual_seed(1))
    table = table.to(torch.int32)[None]
    plan = _c().paged_plan(table, [T], [T], page_size=page, num_pages=T // page, q_heads=H,
                           kv_heads=H, head_dim=D, dtype=dtype, device="cuda:0")
    kd, vd = (torch.zeros(T // page, H, page, D, dtype=dtype, device="cuda:0") for _ in range(2))
    kw = {}
    if rotary:
        kw["cos"], kw["sin"] = _c().rotary_tables(T, rotary, device="cuda:0")
    q = _c().paged_append(x, x, kd, vd, plan, q=x, **kw)
    want = bits.view(T, H, D)[:, :, rotary:]

    def pages(p):
        return p.view(torch.int16).cpu()[table[0].long()].transpose(1, 2).reshape(T, H, D)
    assert torch.equal(pages(vd), bits.view(T, H, D))
    assert torch.equal(pages(kd)[:, :, rotary:], want)
    assert torch.equal(q.view(torch.int16).cpu()[:, :, rotary:], want)
