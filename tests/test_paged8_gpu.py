"""GPU tests of the paged cache of 8 bits against float64 restatements
(tests/paged8_helpers.py, where the tolerances are derived)."""

import pytest
import torch

from tests.paged8_helpers import (BLOCK, attention8_tolerance, empty_pool, fill, filled_pool8,
                                  largest_weight, scale_of, values)
from tests.paged_helpers import EPS, attention64, make_table, rows64, slots_of
from tests.test_paged_gpu import SHAPES

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


def _plan(table, ctx, new, pool, page, Hq, Hkv, D, dtype):
    return _c().paged_plan(table, ctx, new, page_size=page, num_pages=pool, q_heads=Hq,
                           kv_heads=Hkv, head_dim=D, dtype=dtype, device=DEV,
                           cache_dtype=torch.int8)


def _setup(lens, page, dtype, Hq, Hkv, D, seed=0, spread=0):
    table, pool, ctx, new = make_table(lens, page, seed)
    kc, ks = filled_pool8(table, pool, ctx, Hkv, D, page, seed + 1)
    vc, vs = filled_pool8(table, pool, ctx, Hkv, D, page, seed + 5, spread)
    g = torch.Generator().manual_seed(seed + 2)
    q = (1.5 * torch.randn(sum(new), Hq, D, generator=g)).to(dtype)
    return table, pool, ctx, new, kc, ks, vc, vs, _plan(table, ctx, new, pool, page, Hq, Hkv, D,
                                                       dtype), q


def _attend(case, **kw):
    table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
    return _c().paged_attention(q.cuda(), kc.cuda(), vc.cuda(), plan, k_scales=ks.cuda(),
                                v_scales=vs.cuda(), **kw)


def _expected(case, page, scale=None):
    """The outputs in float64, and their bounds."""
    table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
    D = q.shape[-1]
    at = (table, ctx, new, page, D ** -0.5 if scale is None else scale)
    ref, mag, size = attention64(q, values(kc, ks), values(vc, vs), *at)
    largest = largest_weight(q, values(kc, ks), vs, *at)
    return ref, attention8_tolerance(ref, mag, size, largest, D, max(ctx), q.dtype)


def _check(o, case, page, scale=None):
    q = case[-1]
    D = q.shape[-1]
    ref, tol = _expected(case, page, scale)
    err = (o.double().cpu() - ref).abs()
    print(f"[paged8] {q.dtype} D={D} worst {float((err / tol).max()):.3f} of the bound", flush=True)
    assert bool((err <= tol).all()), float((err / tol).max())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_attention_against_float64(hip_device, shape, dtype):
    lens, page, Hq, Hkv, D = shape
    case = _setup(lens, page, dtype, Hq, Hkv, D, seed=len(lens) + D)
    _check(_attend(case), case, page)


WIDE = [([(3900, 512)], 64, 64, 32, 128),              # each split in two
        ([(1100, 340), (2100, 341), (2003, 511), (1500, 171)], 16, 96, 32, 112)]


@pytest.mark.parametrize("shape", WIDE, ids=range(len(WIDE)))
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
def test_tiles_of_256_rows(hip_device, shape, dtype):
    """Three kv heads of them against float64."""
    lens, page, Hq, Hkv, D = shape
    case = _setup(lens, page, dtype, Hq, Hkv, D, seed=3)
    assert case[-2]._info[8] > 0 and case[-2]._info[9] == 0
    heads = [0, 1, Hkv - 1]
    rows = [h * (Hq // Hkv) + i for h in heads for i in range(Hq // Hkv)]
    few = case[:4] + tuple(t[:, heads] for t in case[4:8]) + (None, case[-1][:, rows])
    _check(_attend(case)[:, rows], few, page)


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (32, 2)])
def test_single_tokens_in_the_launch_of_many_rows(hip_device, dtype, D, Hq, Hkv):
    """Both split: rows of a few tokens and of whole tiles."""
    lens = [(3000, 80), (3000, 1), (700, 1), (0, 1), (1500, 24)]
    case = _setup(lens, 64, dtype, Hq, Hkv, D, seed=8)
    info = list(case[-2]._info)
    assert info[6:9] == [0, 0, 0] and info[5] > 1
    _check(_attend(case), case, 64)


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_attention_scale_and_large_scores(hip_device, dtype):
    case = _setup([(100, 20), (700, 1)], 32, dtype, 8, 2, 64, seed=5)
    _check(_attend(case, softmax_scale=1.0), case, 32, scale=1.0)


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", [[(0, 8)] * 40, [(7, 1)] * 200], ids=["many", "few"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_pieces_make_up_their_weight(hip_device, D, lens, dtype):
    """A hundred thousand weights of rows of a few positions and small scores, whose
    bound leaves no room for a weight whose second piece belongs to another rounding
    of it (one in 2^13 lies that near a border)."""
    case = _setup(lens, 16, dtype, 64, 8, D, seed=21)
    _check(_attend(case, softmax_scale=2.0 ** -9), case, 16, scale=2.0 ** -9)


@pytest.mark.parametrize("dtype,spread", [(BF, 3), (BF, 10), (BF, 20), (HF, 3), (HF, 10), (FF, 3),
                                          (FF, 10), (FF, 20)])
@pytest.mark.parametrize("n", [1, 70])
def test_value_blocks_of_any_loudness(hip_device, dtype, spread, n):
    """Scales of neighbouring blocks up to 2^41 apart (fp16's own range is 2^30
    wide), and rows whose weights lie on the quiet ones."""
    case = _setup([(200, n), (90, n)], 32, dtype, 4, 2, 64, seed=8, spread=spread)
    table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
    for s in range(2):                 # the louder half of the blocks: keys of tiny scores
        for b in range(-(-ctx[s] // BLOCK)):
            page, j = int(table[s, b * BLOCK // 32]), b % 2
            for h in range(2):
                if vs[page, h, j] > vs[int(table[s, 0]), h, 0]:
                    kc[page, h, j * BLOCK:(j + 1) * BLOCK] = 0
    q *= 4
    _check(_attend(case), case, 32)


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_blocks_of_zeros_and_of_the_smallest_scale_count(hip_device, dtype):
    """Values of zero have weights all the same; keys of the smallest scale have
    scores of (nearly) zero."""
    for n in (1, 40):
        case = _setup([(100, n)], 16, dtype, 4, 2, 64, seed=4)
        table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
        for b in (0, 3):
            vc[int(table[0, b])] = 0
            vs[int(table[0, b])] = 2.0 ** -126
            ks[int(table[0, b + 1])] = 2.0 ** -126
        vs[int(table[0, 2])] = 0.0
        ks[int(table[0, 2])] = 0.0
        _check(_attend(case), case, 16)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [3, 60])
def test_blocks_that_are_not_numbers(hip_device, dtype, D, n):
    """A row that sees a position of a block whose scale is NaN is NaN, the others keep
    their bound."""
    case = _setup([(37, n), (64, n)], 16, dtype, 4, 2, D, seed=9)
    table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
    first = [c - m for c, m in zip(ctx, new)]
    bad = (first[0] + n // 2 + 15) // 16             # (no token sees it for n 3)
    if bad * 16 < ctx[0]:
        vs[int(table[0, bad]), 1, 0] = float("nan")
    last = (ctx[1] - 1) // 16
    ks[int(table[1, last]), 0, 0] = float("nan")
    o = _attend(case).cpu()
    ok_v, ok_k = vs.clone(), ks.clone()
    ok_v[torch.isnan(ok_v)] = 1.0
    ok_k[torch.isnan(ok_k)] = 1.0
    ref, tol = _expected((table, pool, ctx, new, kc, ok_k, vc, ok_v, plan, q), 16)
    sees_v = torch.zeros(2 * n, 4, dtype=torch.bool)
    sees_k = torch.zeros(2 * n, 4, dtype=torch.bool)
    for i in range(n):
        sees_v[i, 2:] = first[0] + i >= bad * 16
        sees_k[n + i, :2] = first[1] + i >= last * 16
    lost = (sees_v | sees_k)[..., None].expand_as(o)
    assert bool(torch.isnan(o[lost]).all())
    assert bool(((o.double() - ref).abs() <= tol)[~lost].all())


def test_attention_strides_rows_behind_and_out(hip_device):
    for dtype in (BF, FF):
        case = _setup([(50, 3), (9, 30)], 32, dtype, 8, 2, 128, seed=2)
        table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
        T = q.shape[0]
        want = _attend(case)
        pools = dict(k_pages=kc.cuda(), v_pages=vc.cuda(), k_scales=ks.cuda(), v_scales=vs.cuda())
        wide = torch.full((T + 4, 8 + 5, 128), float("nan"), dtype=dtype, device=DEV)
        wide[:T, 2:10] = q.cuda()
        got = _c().paged_attention(wide[:, 2:10], plan=plan, **pools)
        assert torch.equal(got[:T], want) and bool((got[T:] == 0).all())
        out = torch.full((T + 4, 8, 128), 7.0, dtype=dtype, device=DEV)
        assert _c().paged_attention(wide[:, 2:10], plan=plan, out=out, **pools) is out
        assert torch.equal(out[:T], want) and bool((out[T:] == 7).all())
        odd = torch.empty(T * 8 * 128 + 1, dtype=dtype, device=DEV)
        odd[1:] = q.cuda().flatten()
        assert torch.equal(_c().paged_attention(odd[1:].view(T, 8, 128), plan=plan, **pools), want)


def test_offsets_past_32_bits(hip_device):
    """Pages whose byte offsets pass 2^32: append, then attention."""
    page, Hkv, D = 256, 8, 128
    pool = (1 << 32) // (page * Hkv * D) + 40
    kd = torch.zeros(pool, Hkv, page, D, dtype=torch.int8, device=DEV)
    vd = torch.zeros_like(kd)
    ksd = torch.zeros(pool, Hkv, page // 16, device=DEV)
    vsd = torch.zeros_like(ksd)
    lens = [(0, 700), (0, 340)]
    table = torch.tensor([[pool - 1, 3, pool - 7], [pool - 2, 11, -1]], dtype=torch.int32)
    ctx = new = [700, 340]
    plan = _plan(table, ctx, new, pool, page, 16, Hkv, D, BF)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1040, Hkv, D, generator=g).to(BF) for _ in range(2))
    _c().paged_append(k.cuda(), v.cuda(), kd, vd, plan, k_scales=ksd, v_scales=vsd)
    pages = table[table >= 0].long().cuda()
    small = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32)
    kc, ks = empty_pool(5, Hkv, page, D, 1)
    vc, vs = empty_pool(5, Hkv, page, D, 2)
    slots = slots_of(small, ctx, new, page)
    fill(kc, ks, k.double(), slots, [0] * 1040)
    fill(vc, vs, v.double(), slots, [0] * 1040)
    for c, s, dc, ds in ((kc, ks, kd, ksd), (vc, vs, vd, vsd)):
        got, gs = dc[pages].cpu(), ds[pages].cpu()
        for p, off, _ in slots:
            assert torch.equal(got[p, :, off], c[p, :, off])
            assert torch.equal(gs[p, :, off // 16], s[p, :, off // 16])
    new2 = [1, 40]
    plan = _plan(table, ctx, new2, pool, page, 16, Hkv, D, BF)
    q = torch.randn(41, 16, D, generator=g).to(BF)
    o = _c().paged_attention(q.cuda(), kd, vd, plan, k_scales=ksd, v_scales=vsd)
    case = (small, 5, ctx, new2, kc, ks, vc, vs, plan, q)
    _check(o, case, page)


def test_streams_graphs_and_repeats(hip_device):
    """On a stream of its own, captured (several replays between eager calls), and two
    graphs with a workspace each: the bits of the first call."""
    case = _setup([(3000, 1), (800, 20), (40, 1)], 64, BF, 8, 2, 128, seed=6)
    table, pool, ctx, new, kc, ks, vc, vs, plan, q = case
    x = dict(k_pages=kc.cuda(), v_pages=vc.cuda(), k_scales=ks.cuda(), v_scales=vs.cuda())
    qd = q.cuda()
    call = lambda: _c().paged_attention(qd, plan=plan, **x)          # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
    torch.cuda.current_stream().wait_stream(side)
    plan.wait()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        assert torch.equal(call(), want)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _rows(new, Hq, Hkv, D, dtype, seed, loud=3.0):
    """One projection's rows, some tokens louder than others."""
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    x = torch.randn(T, Hq + 2 * Hkv, D, generator=g)
    x *= 2.0 ** (loud * (torch.rand(T, 1, 1, generator=g) - 0.5))
    x = x.to(dtype)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


APPENDS = [
    # lens, page, Hq, Hkv, D, rotary, interleaved, norm
    ([(0, 1)], 16, 4, 2, 64, 64, False, True),
    ([(15, 1), (16, 1), (31, 2), (40, 5)], 16, 4, 2, 128, 128, False, True),
    ([(0, 16), (3, 13), (5, 40), (100, 0)], 32, 8, 2, 128, 64, True, False),
    ([(9, 70), (14, 3)], 64, 6, 3, 80, 32, False, True),
    ([(9, 70), (14, 3)], 128, 2, 1, 16, 16, True, True),
    ([(130, 33), (255, 2)], 256, 4, 4, 256, 256, False, True),
    ([(1, 17), (0, 1), (7, 1)], 16, 5, 5, 96, 96, True, False),
    ([(30, 50), (64, 1)], 64, 4, 2, 192, 0, False, True),
    ([(30, 50), (64, 1)], 64, 4, 2, 112, 0, False, False),
]


@pytest.mark.parametrize("shape", APPENDS, ids=range(len(APPENDS)))
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_append_against_float64(hip_device, shape, dtype):
    """Codes and scales are those of the definition (keys are formed in fp64, whose
    rounding stays far from a border of these inputs); queries are
    paged_append's bits into pages of the model's type; the rest is untouched."""
    lens, page, Hq, Hkv, D, rot, inter, norm = shape
    table, pool, ctx, new = make_table(lens, page, 7)
    before = [c - n for c, n in zip(ctx, new)]
    kc, ks = filled_pool8(table, pool, before, Hkv, D, page, 11)
    vc, vs = filled_pool8(table, pool, before, Hkv, D, page, 12)
    q, k, v = _rows(new, Hq, Hkv, D, dtype, 13)
    g = torch.Generator().manual_seed(14)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None
              for _ in range(2))
    cos = sin = None
    if rot:
        cos, sin = _c().rotary_tables(max(ctx), rot, device="cpu")
    dev = lambda t: None if t is None else t.cuda()                  # noqa: E731
    plan = _plan(table, ctx, new, pool, page, Hq, Hkv, D, dtype)
    kd, ksd, vd, vsd = (t.cuda() for t in (kc, ks, vc, vs))
    qkv = torch.cat([q, k, v], 1).cuda()
    kw = dict(cos=dev(cos), sin=dev(sin), interleaved=inter, q_norm=dev(wq), k_norm=dev(wk))
    got = _c().paged_append(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], kd, vd, plan, q=qkv[:, :Hq],
                            k_scales=ksd, v_scales=vsd, **kw)
    slots = slots_of(table, ctx, new, page)
    pos = torch.tensor([p for _, _, p in slots])
    at = (None, None) if cos is None else (cos[pos], sin[pos])
    held = [c - n for c, n in zip(ctx, new) for _ in range(n)]
    fill(kc, ks, rows64(k, wk, *at, inter), slots, held)
    fill(vc, vs, v.double(), slots, held)
    for a, b in ((kd, kc), (vd, vc)):
        assert torch.equal(a.cpu(), b)
    for a, b in ((ksd, ks), (vsd, vs)):
        assert torch.equal(a.cpu().view(torch.int32), b.view(torch.int32))
    plain = _c().paged_plan(table, ctx, new, page_size=page, num_pages=pool, q_heads=Hq,
                            kv_heads=Hkv, head_dim=D, dtype=dtype, device=DEV)
    pages = [torch.empty(pool, Hkv, page, D, dtype=dtype, device=DEV) for _ in range(2)]
    want = _c().paged_append(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], *pages, plain,
                             q=qkv[:, :Hq], **kw)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, FF], ids=["bf16", "f32"])
def test_a_block_filled_token_by_token(hip_device, dtype):
    """Forty steps of one token, each louder or quieter than the last: the definition's
    codes at every step, and every value within one final scale of its own."""
    page, Hkv, D, steps = 32, 2, 64, 40
    table, pool, _, _ = make_table([(0, steps)], page, 1)
    kc, ks = empty_pool(pool, Hkv, page, D, 1)
    vc, vs = empty_pool(pool, Hkv, page, D, 2)
    kd, ksd, vd, vsd = (t.cuda() for t in (kc, ks, vc, vs))
    g = torch.Generator().manual_seed(3)
    rows = [(torch.randn(2, 1, Hkv, D, generator=g) * 1.17 ** i / (1 + i % 3)).to(dtype)
            for i in range(steps)]
    for i, (k, v) in enumerate(rows):
        plan = _plan(table, [i + 1], [1], pool, page, 4, Hkv, D, dtype)
        _c().paged_append(k.cuda(), v.cuda(), kd, vd, plan, k_scales=ksd, v_scales=vsd)
        slots = slots_of(table, [i + 1], [1], page)
        fill(kc, ks, k.double(), slots, [i])
        fill(vc, vs, v.double(), slots, [i])
        for a, b in ((kd, kc), (vd, vc), (ksd, ks), (vsd, vs)):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)), i
    for which, (codes, scales) in enumerate(((kc, ks), (vc, vs))):
        x = values(codes, scales)
        for i in range(steps):
            p, off = int(table[0, i // page]), i % page
            s = scales[p, :, off // BLOCK].double()[:, None]
            assert bool(((x[p, :, off] - rows[i][which][0].double()).abs() <= s).all())


def test_borders_zeros_and_the_ends_of_the_range(hip_device):
    """Largest values next to 127 scales, quotients half-way between codes, zeros, and
    fp32's largest and smallest numbers."""
    cases = [127.0, 127.0 * (1 + 2.0 ** -23), 63.5, 0.0, 1e-45, 2.0 ** -126, 3.4e38, 1e-38, 254.0]
    table, pool, ctx, new = make_table([(0, 16 * len(cases))], 16, 1)
    k = torch.zeros(16 * len(cases), 1, 32)
    for i, top in enumerate(cases):
        s = scale_of(top)
        # ties of both kinds, as far as they stay below the largest
        ties = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -125.5, 0.25, 62.5], dtype=FF)
        x = (ties.double() * s).clamp(-top, top).to(FF)
        k[16 * i + 3, 0, :9] = x
        k[16 * i + 7, 0, 31] = top if i % 2 else -top
    plan = _plan(table, ctx, new, pool, 16, 1, 1, 32, FF)
    kc, ks = empty_pool(pool, 1, 16, 32, 1)
    vc, vs = empty_pool(pool, 1, 16, 32, 2)
    kd, ksd, vd, vsd = (t.cuda() for t in (kc, ks, vc, vs))
    _c().paged_append(k.cuda(), (-k).cuda(), kd, vd, plan, k_scales=ksd, v_scales=vsd)
    slots = slots_of(table, ctx, new, 16)
    fill(kc, ks, k.double(), slots, [0] * len(k))
    fill(vc, vs, -k.double(), slots, [0] * len(k))
    for a, b in ((kd, kc), (vd, vc), (ksd, ks), (vsd, vs)):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_values_that_are_not_finite(hip_device, dtype):
    """An infinity or a NaN makes its block's scale NaN and no other's; what follows
    in the block leaves it so, and a block that starts anew is a number again."""
    page, Hkv, D = 16, 2, 64
    table, pool, ctx, new = make_table([(0, 40)], page, 1)
    kd, ksd, vd, vsd = (t.cuda() for t in (*empty_pool(pool, Hkv, page, D, 1),
                                           *empty_pool(pool, Hkv, page, D, 2)))
    q, k, v = _rows(new, 4, Hkv, D, dtype, 5)
    k[20, 1, 7], v[36, 0, 63] = float("inf"), float("nan")
    cos, sin = _c().rotary_tables(64, D, device=DEV)
    args = dict(k_scales=ksd, v_scales=vsd, cos=cos, sin=sin)
    plan = _plan(table, ctx, new, pool, page, 4, Hkv, D, dtype)
    _c().paged_append(k.cuda(), v.cuda(), kd, vd, plan, **args)
    t = table[0].long()
    bad_k = torch.isnan(ksd[t[:3].cuda(), :, 0]).cpu().tolist()
    bad_v = torch.isnan(vsd[t[:3].cuda(), :, 0]).cpu().tolist()
    assert bad_k == [[False, False], [False, True], [False, False]]
    assert bad_v == [[False, False], [False, False], [True, False]]
    one = torch.ones(1, Hkv, D, dtype=dtype, device=DEV)
    for context, nan in ((41, True), (33, False)):       # (33: its first position again)
        plan = _plan(table, [context], [1], pool, page, 4, Hkv, D, dtype)
        _c().paged_append(one, one, kd, vd, plan, **args)
        assert torch.isnan(vsd[int(t[2]), :, 0]).cpu().tolist() == [nan, False]


def test_append_calls_that_are_refused(hip_device):
    C = _c()
    table, pool, ctx, new = make_table([(20, 2)], 32, 1)
    plan = _plan(table, ctx, new, pool, 32, 4, 2, 64, BF)
    pages = [torch.zeros(pool, 2, 32, 64, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(pool, 2, 2, device=DEV) for _ in range(2)]
    k = torch.zeros(2, 2, 64, dtype=BF, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=BF, device=DEV)

    def append(kp=pages[0], ks=scales[0], vs=scales[1], p=plan):
        return C.paged_append(k, k.clone(), kp, pages[1], p, k_scales=ks, v_scales=vs)

    def attend(kp=pages[0], ks=scales[0], vs=scales[1], p=plan):
        return C.paged_attention(q, kp, pages[1], p, k_scales=ks, v_scales=vs)
    for call in (append, attend):
        call()
        with pytest.raises(RuntimeError, match="need k_scales and v_scales"):
            call(ks=None)
        with pytest.raises(RuntimeError, match="v_scales must be a contiguous"):
            call(vs=scales[1][:, :1])
        with pytest.raises(RuntimeError, match="k_scales must be a contiguous"):
            call(ks=scales[0].half())
        with pytest.raises(RuntimeError, match="k_pages must be a contiguous"):
            call(kp=pages[0].to(BF))
        with pytest.raises(RuntimeError, match="inference only"):
            call(ks=scales[0].clone().requires_grad_())
    with pytest.raises(RuntimeError, match="k_scales and v_scales must be two"):
        append(vs=scales[0])
    plain = C.paged_plan(table, ctx, new, page_size=32, num_pages=pool, q_heads=4, kv_heads=2,
                         head_dim=64, dtype=BF, device=DEV)
    wide = torch.zeros(pool, 2, 32, 64, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="belong to pages of int8"):
        C.paged_attention(q, wide, wide.clone(), plain, k_scales=scales[0], v_scales=scales[1])
    with pytest.raises(RuntimeError, match="k_pages must be a contiguous"):
        C.paged_attention(q, pages[0], pages[1], plain)


def test_a_step_of_no_tokens(hip_device):
    table, pool, ctx, new = make_table([(20, 0), (3, 0)], 32, 1)
    plan = _plan(table, ctx, new, pool, 32, 4, 2, 64, BF)
    pages = [torch.zeros(pool, 2, 32, 64, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = dict(k_scales=torch.zeros(pool, 2, 2, device=DEV),
                  v_scales=torch.zeros(pool, 2, 2, device=DEV))
    k = torch.zeros(0, 2, 64, dtype=BF, device=DEV)
    q = torch.zeros(3, 4, 64, dtype=BF, device=DEV)
    assert _c().paged_append(k, k, *pages, plan, **scales) is None
    assert bool((_c().paged_attention(q, *pages, plan, **scales) == 0).all())


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [48, 128])
def test_append_of_rows_at_any_alignment_and_in_place(hip_device, D, dtype):
    """Rows whose strides are no whole vectors give the codes of contiguous ones; queries
    may be turned where they lie."""
    page, Hq, Hkv = 32, 4, 2
    table, pool, ctx, new = make_table([(7, 30), (40, 1)], page, 3)
    T = sum(new)
    q, k, v = _rows(new, Hq, Hkv, D, dtype, 9)
    cos, sin = _c().rotary_tables(max(ctx), 32, device=DEV)
    weights = torch.rand(2, D, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    kw = dict(cos=cos, sin=sin, q_norm=weights[0], k_norm=weights[1])
    plan = _plan(table, ctx, new, pool, page, Hq, Hkv, D, dtype)
    pools = [t.cuda() for t in (*filled_pool8(table, pool, ctx, Hkv, D, page, 1),
                                *filled_pool8(table, pool, ctx, Hkv, D, page, 2))]

    def append(q, k, v, q_out=None):
        kc, ks, vc, vs = (t.clone() for t in pools)
        got = _c().paged_append(k, v, kc, vc, plan, q=q, q_out=q_out, k_scales=ks, v_scales=vs,
                                **kw)
        return got.clone(), kc, ks, vc, vs

    want = append(q.cuda(), k.cuda(), v.cuda())
    odd = torch.full((T + 2, (Hq + 2 * Hkv) * D + 3), float("nan"), dtype=dtype, device=DEV)
    rows = odd[:T, 1:1 + (Hq + 2 * Hkv) * D].unflatten(1, (-1, D))
    rows.copy_(torch.cat([q, k, v], 1))
    got = append(rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:])
    place = q.cuda().contiguous()
    there = append(place, k.cuda(), v.cuda(), q_out=place)
    for a, b, c in zip(want, got, there):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
