"""GPU tests of the paged cache's append and attention against float64
restatements (tests/paged_helpers.py, where the tolerances are derived)."""

import numpy as np
import pytest
import torch

from tests.paged_helpers import (EPS, attention64, attention_tolerance, filled_pool, make_table,
                                 rows64, slots_of)

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


def _setup(lens, page_size, dtype, Hq, Hkv, D, seed=0):
    table, pool, ctx, new = make_table(lens, page_size, seed)
    kp, vp = filled_pool(table, pool, ctx, Hkv, D, page_size, dtype, seed + 1)
    plan = _c().paged_plan(table, ctx, new, page_size=page_size, num_pages=pool, q_heads=Hq,
                           kv_heads=Hkv, head_dim=D, dtype=dtype, device="cuda:0")
    g = torch.Generator().manual_seed(seed + 2)
    q = (1.5 * torch.randn(sum(new), Hq, D, generator=g)).to(dtype)
    return table, pool, ctx, new, kp, vp, plan, q


def _attend(case, **kw):
    table, pool, ctx, new, kp, vp, plan, q = case
    return _c().paged_attention(q.cuda(), kp.cuda(), vp.cuda(), plan, **kw)


def _check(o, case, page_size, scale=None):
    table, pool, ctx, new, kp, vp, plan, q = case
    D = q.shape[-1]
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, page_size,
                                 D ** -0.5 if scale is None else scale)
    tol = attention_tolerance(ref, mag, size, D, max(ctx), q.dtype)
    err = (o.double().cpu() - ref).abs()
    print(f"[paged] {q.dtype} D={D} worst {float((err / tol).max()):.3f} of the bound", flush=True)
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [
    # one token, one position; a tile's borders; a page's borders
    ([(0, 1)], 16, 4, 2, 64),
    ([(15, 1), (16, 1), (31, 1), (32, 1), (63, 1), (64, 1)], 16, 4, 2, 64),
    ([(0, 5), (3, 2), (30, 3)], 32, 8, 2, 128),
    # rows of 16, 17, 32, 33, 64, 65 and 128, 129 to a kv head
    ([(40, 16), (7, 17), (0, 32), (100, 33)], 64, 2, 2, 64),
    ([(9, 64), (70, 65)], 128, 2, 2, 128),
    ([(5, 128), (33, 129)], 256, 1, 1, 64),
    # heads: groups of 3, 5, 20; more than 16 rows from one token
    ([(77, 1), (200, 7)], 32, 6, 2, 128),
    ([(50, 3), (300, 1)], 16, 20, 4, 96),
    ([(129, 1), (0, 2)], 32, 20, 1, 128),
    ([(500, 1)], 64, 48, 1, 64),
    # head dims that fill no instance, and the largest
    ([(33, 9), (70, 1)], 16, 4, 2, 16),
    ([(33, 70), (70, 1)], 16, 4, 2, 80),
    ([(100, 40), (64, 1)], 32, 4, 2, 112),
    ([(90, 30), (64, 1), (0, 20)], 32, 4, 2, 192),
    ([(90, 80), (64, 1), (0, 20)], 64, 4, 1, 256),
    # a sequence that sits the step out, contexts that are split
    ([(20, 0), (3000, 1), (5, 1)], 64, 8, 2, 128),
    ([(2500, 40), (9, 1)], 64, 8, 2, 64),
    ([(1800, 5)], 128, 14, 2, 128),
]


@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_attention_against_float64(hip_device, shape, dtype):
    lens, page, Hq, Hkv, D = shape
    case = _setup(lens, page, dtype, Hq, Hkv, D, seed=len(lens) + D)
    _check(_attend(case), case, page)


@pytest.mark.parametrize("dtype", [BF, FF], ids=["bf16", "f32"])
def test_attention_scale_and_large_scores(hip_device, dtype):
    case = _setup([(100, 20), (700, 1)], 32, dtype, 8, 2, 64, seed=5)
    _check(_attend(case, softmax_scale=1.0), case, 32, scale=1.0)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [3, 60])
def test_what_a_token_does_not_see_does_not_reach_it(hip_device, dtype, D, n):
    """Infinities and NaN in keys and values of later tokens: rows that do not
    see them keep their bits' bound, rows that do carry them."""
    case = _setup([(37, n), (64, n)], 16, dtype, 4, 2, D, seed=9)
    table, pool, ctx, new, kp, vp, plan, q = case
    bad = n // 2                                     # new token of sequence 0
    pos = ctx[0] - n + bad
    vp[int(table[0, pos // 16]), 1, pos % 16, 5] = float("inf")
    vp[int(table[0, pos // 16]), 1, pos % 16, 6] = float("nan")
    pos2 = ctx[1] - 1                                # the last token of sequence 1
    kp[int(table[1, pos2 // 16]), 0, pos2 % 16, 3] = float("nan")
    o = _attend(case).cpu()
    ref, mag, size = attention64(q, kp, vp, table, ctx, new, 16, D ** -0.5)
    tol = attention_tolerance(ref, mag, size, D, max(ctx), dtype)
    fine = torch.isfinite(ref)
    assert bool(((o.double() - ref).abs() <= tol)[fine].all())
    assert fine[:bad].all() and not fine[bad:n, 2:, 5].any()
    assert bool((o[bad:n, 2:, 5] == float("inf")).all())
    assert bool(torch.isnan(o[bad:n, 2:, 6]).all())
    assert bool(torch.isnan(o[2 * n - 1, :2]).all())
    assert bool(torch.isfinite(o[n:2 * n - 1]).all())


def test_attention_strides_rows_behind_and_out(hip_device):
    case = _setup([(50, 3), (9, 30)], 32, BF, 8, 2, 128, seed=2)
    table, pool, ctx, new, kp, vp, plan, q = case
    T = q.shape[0]
    want = _attend(case)
    kd, vd = kp.cuda(), vp.cuda()
    wide = torch.full((T + 4, 8 + 5, 128), float("nan"), dtype=BF, device="cuda:0")
    wide[:T, 2:10] = q.cuda()
    got = _c().paged_attention(wide[:, 2:10], kd, vd, plan)
    assert torch.equal(got[:T], want) and bool((got[T:] == 0).all())
    out = torch.full((T + 4, 8, 128), 7.0, dtype=BF, device="cuda:0")
    assert _c().paged_attention(wide[:, 2:10], kd, vd, plan, out=out) is out
    assert torch.equal(out[:T], want) and bool((out[T:] == 7).all())
    # a view that starts off a 16-byte border
    odd = torch.empty(T * 8 * 128 + 1, dtype=BF, device="cuda:0")
    odd[1:] = q.cuda().flatten()
    assert torch.equal(_c().paged_attention(odd[1:].view(T, 8, 128), kd, vd, plan), want)


def test_offsets_past_32_bits(hip_device):
    """Pages whose element offsets pass 2^31 (and byte offsets 2^32)."""
    page, Hkv, D = 256, 8, 128
    pool = (1 << 31) // (page * Hkv * D) + 40
    kd = torch.zeros(pool, Hkv, page, D, dtype=BF, device="cuda:0")
    vd = torch.zeros_like(kd)
    lens = [(700, 1), (300, 40)]
    table, _, ctx, new = make_table(lens, page, 1)
    pages = torch.tensor([[pool - 1, 3, pool - 7], [pool - 2, 11, -1]], dtype=torch.int32)
    small, _, _, _ = make_table(lens, page, 1)
    small_pool = [torch.randn(5, Hkv, page, D, generator=torch.Generator().manual_seed(i)).to(BF)
                  for i in (1, 2)]
    small = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32)
    for i, p in enumerate((pool - 1, 3, pool - 7, pool - 2, 11)):
        kd[p], vd[p] = small_pool[0][i].cuda(), small_pool[1][i].cuda()
    q = torch.randn(41, 16, D, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    kw = dict(page_size=page, q_heads=16, kv_heads=Hkv, head_dim=D, device="cuda:0")
    a = _c().paged_plan(pages, ctx, new, num_pages=pool, **kw)
    b = _c().paged_plan(small, ctx, new, num_pages=5, **kw)
    ks, vs = small_pool[0].cuda(), small_pool[1].cuda()
    assert torch.equal(_c().paged_attention(q, kd, vd, a), _c().paged_attention(q, ks, vs, b))
    k = torch.randn(41, Hkv, D, device="cuda:0").to(BF)
    _c().paged_append(k, -k, kd, vd, a)
    for t, (p, o, _) in enumerate(slots_of(pages, ctx, new, page)):
        assert torch.equal(kd[p, :, o], k[t]) and torch.equal(vd[p, :, o], -k[t])


# ----------------------------------------------------------------- append
def _append_case(lens, page, dtype, Hq, Hkv, D, rot, interleaved, norm, seed, norm_dtype=None):
    table, pool, ctx, new = make_table(lens, page, seed)
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(dtype)
    kp = torch.randn(pool, Hkv, page, D, generator=g).to(dtype)
    vp = torch.randn(pool, Hkv, page, D, generator=g).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(norm_dtype or dtype) for _ in range(2)]
    w = w if norm else [None, None]
    cs = (None, None)
    if rot:
        cs = _c().rotary_tables(max(ctx), rot, device="cpu")
    plan = _c().paged_plan(table, ctx, new, page_size=page, num_pages=pool, q_heads=Hq,
                           kv_heads=Hkv, head_dim=D, dtype=dtype, device="cuda:0")
    return table, ctx, new, qkv, kp, vp, w, cs, plan


def _rows_tolerance(ref, x, w, dtype, rot, norm):
    """Half a step of the output; fp32: a rotated channel is two products and a
    sum (3 roundings of a pair's size), a norm adds the sum of D squares, the root,
    the quotient and two products ((D + 8) 2^-24 relative, halved by the root)."""
    u = 2.0 ** -24
    size = ref.abs().amax(-1, keepdim=True)
    return EPS[dtype] / 2 * ref.abs() + u * (3 * rot + (norm and (x.shape[-1] + 8))) * 2 * size


APPENDS = [
    ([(0, 1)], 16, 4, 2, 64, 64, False, True),
    ([(1000, 1), (15, 1), (16, 1)], 16, 8, 2, 128, 128, False, False),
    ([(5, 40), (0, 0), (31, 2), (0, 1)], 32, 6, 3, 128, 128, False, True),
    ([(3, 70)], 64, 12, 12, 64, 32, True, False),
    ([(3, 70)], 64, 4, 4, 80, 32, False, True),
    ([(9, 9), (0, 5)], 128, 4, 1, 96, 96, True, True),
    ([(9, 9), (0, 5)], 256, 4, 1, 256, 256, False, True),
    ([(2, 6)], 16, 2, 2, 16, 16, False, True),
    ([(2, 6)], 16, 2, 2, 208, 0, False, True),
    ([(2, 6), (100, 7)], 16, 3, 1, 112, 48, True, False),
]


@pytest.mark.parametrize("shape", APPENDS, ids=range(len(APPENDS)))
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
def test_append_against_float64(hip_device, shape, dtype):
    lens, page, Hq, Hkv, D, rot, inter, norm = shape
    table, ctx, new, qkv, kp, vp, w, cs, plan = _append_case(lens, page, dtype, Hq, Hkv, D, rot,
                                                             inter, norm, seed=D + rot)
    T = sum(new)
    dev = "cuda:0"
    x = qkv.to(dev)
    kd, vd = kp.to(dev), vp.to(dev)
    on = lambda t: None if t is None else t.to(dev)      # noqa: E731
    q = _c().paged_append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], kd, vd, plan, q=x[:, :Hq],
                          cos=on(cs[0]), sin=on(cs[1]), interleaved=inter, q_norm=on(w[0]),
                          k_norm=on(w[1]))
    places = slots_of(table, ctx, new, page)
    pos = torch.tensor([p[2] for p in places])
    cos, sin = (None, None) if not rot else (cs[0][pos], cs[1][pos])
    for got, src, wt in ((q, qkv[:, :Hq], w[0]), (None, qkv[:, Hq:Hq + Hkv], w[1])):
        ref = rows64(src, wt, cos, sin, inter)
        if got is None:
            got = torch.stack([kd[p, :, o] for p, o, _ in places])
        tol = _rows_tolerance(ref, src, wt, dtype, bool(rot), norm)
        assert bool(((got.double().cpu() - ref).abs() <= tol).all())
    # values bit for bit; every other slot as it was
    kw, vw = kd.cpu(), vd.cpu()
    for t, (p, o, _) in enumerate(places):
        assert torch.equal(vw[p, :, o], qkv[t, Hq + Hkv:])
        kw[p, :, o], vw[p, :, o] = kp[p, :, o], vp[p, :, o]
    assert torch.equal(kw, kp) and torch.equal(vw, vp)
    assert q.shape == (T, Hq, D)


def test_append_without_queries_and_plain(hip_device):
    """No norm, no rotation: keys bit for bit; strides off the vector border take
    the element loads and give the same."""
    table, ctx, new, qkv, kp, vp, _, _, plan = _append_case([(3, 20), (64, 1)], 32, BF, 4, 2, 64,
                                                            0, False, False, 4)
    x = qkv.cuda()
    kd, vd = kp.cuda(), vp.cuda()
    k, v = x[:, 4:6], x[:, 6:]
    assert _c().paged_append(k, v, kd, vd, plan) is None
    for t, (p, o, _) in enumerate(slots_of(table, ctx, new, 32)):
        assert torch.equal(kd[p, :, o], k[t]) and torch.equal(vd[p, :, o], v[t])
    ke, ve = kp.cuda(), vp.cuda()
    odd = torch.zeros(21, 2, 67, dtype=BF, device="cuda:0")
    odd[..., 1:65] = k
    _c().paged_append(odd[..., 1:65], v, ke, ve, plan)
    assert torch.equal(ke, kd) and torch.equal(ve, vd)


def test_append_in_place_norm_types_and_rows_behind(hip_device):
    args = _append_case([(3, 20), (64, 1)], 32, BF, 4, 2, 64, 64, False, True, 6, torch.float32)
    table, ctx, new, qkv, kp, vp, w, cs, plan = args
    x = qkv.cuda()
    kd, vd = kp.cuda(), vp.cuda()
    kw = dict(cos=cs[0].cuda(), sin=cs[1].cuda(), q_norm=w[0].cuda(), k_norm=w[1].cuda())
    q = torch.cat([x[:, :4], torch.full((3, 4, 64), 5.0, dtype=BF, device="cuda:0")])
    k, v = x[:, 4:6], x[:, 6:]
    want = _c().paged_append(k, v, kd, vd, plan, q=q, **kw)
    assert bool((want[21:] == 0).all())
    ref = rows64(qkv[:, :4], w[0], *(c[torch.tensor([p[2] for p in slots_of(table, ctx, new, 32)])]
                                     for c in cs), False)
    assert bool(((want[:21].double().cpu() - ref).abs()
                 <= _rows_tolerance(ref, ref, None, BF, True, True)).all())
    assert _c().paged_append(k, v, kd, vd, plan, q=q, q_out=q, **kw) is q
    assert torch.equal(q[:21], want[:21]) and bool((q[21:] == 5).all())


def test_far_positions(hip_device):
    """Angles of far positions: the tables hold fp32 of the float64 angle's cosine."""
    cos, sin = _c().rotary_tables(131073, 64, base=500000.0, device="cuda:0")
    i = torch.arange(32, dtype=torch.float64)
    ang = 131072 * 500000.0 ** (-i / 32)
    assert float((cos[131072].double().cpu() - ang.cos()).abs().max()) <= 2.0 ** -24
    assert float((sin[131072].double().cpu() - ang.sin()).abs().max()) <= 2.0 ** -24


# --------------------------------------------- streams, graphs, refusals
def test_another_stream(hip_device):
    case = _setup([(50, 3), (3000, 1)], 32, BF, 8, 2, 128, seed=3)
    table, pool, ctx, new, kp, vp, _, q = case
    want = _attend(case)
    kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    plan = _c().paged_plan(table, ctx, new, page_size=32, num_pages=pool, q_heads=8, kv_heads=2,
                           head_dim=128, device="cuda:0")
    with torch.cuda.stream(s):
        got = _c().paged_attention(qd, kd, vd, plan)
    del plan
    s.synchronize()
    assert torch.equal(got, want)


def test_two_captured_graphs(hip_device):
    """A captured append and attention replays with new inputs; two graphs with
    split contexts keep their partials apart when they run at once."""
    cases = [_setup([(2500, 1), (40, 2)], 64, BF, 8, 2, 128, seed=i) for i in (11, 12)]
    runs = []
    for table, pool, ctx, new, kp, vp, plan, q in cases:
        kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
        k, v = torch.randn(3, 2, 128, device="cuda:0").to(BF), torch.randn(3, 2, 128, device="cuda:0").to(BF)
        cos, sin = _c().rotary_tables(max(ctx), 128, device="cuda:0")
        plan.wait()

        def step(k=k, v=v, kd=kd, vd=vd, plan=plan, qd=qd, cos=cos, sin=sin):
            r = _c().paged_append(k, v, kd, vd, plan, q=qd, cos=cos, sin=sin)
            return _c().paged_attention(r, kd, vd, plan)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        runs.append((graph, out, step, qd, k))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        want = []
        for graph, out, step, qd, k in runs:
            qd.normal_()
            k.normal_()
            want.append(step().clone())
        torch.cuda.synchronize()
        for (graph, out, *_), s in zip(runs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, out, *_), w in zip(runs, want):
            assert torch.equal(out, w)


def test_capture_needs_a_settled_plan(hip_device):
    case = _setup([(20, 1)], 32, BF, 4, 2, 64, seed=3)
    table, pool, ctx, new, kp, vp, plan, q = case
    kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="wait"):
            _c().paged_attention(qd, kd, vd, plan)
        torch.zeros(1, device="cuda:0")


def test_refusals_on_device(hip_device):
    case = _setup([(20, 2)], 32, BF, 4, 2, 64, seed=3)
    table, pool, ctx, new, kp, vp, plan, q = case
    C = _c()
    kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
    with pytest.raises(RuntimeError, match="k_pages must be a contiguous"):
        C.paged_attention(qd, kd[1:], vd, plan)
    with pytest.raises(RuntimeError, match="v_pages must be a contiguous"):
        C.paged_attention(qd, kd, vd.half(), plan)
    with pytest.raises(RuntimeError, match="q must be"):
        C.paged_attention(qd[:1], kd, vd, plan)
    with pytest.raises(RuntimeError, match="q must be"):
        C.paged_attention(qd.float(), kd, vd, plan)
    with pytest.raises(RuntimeError, match="channels must be contiguous"):
        C.paged_attention(qd.transpose(1, 2).contiguous().transpose(1, 2), kd, vd, plan)
    with pytest.raises(RuntimeError, match="inference only"):
        C.paged_attention(qd.clone().requires_grad_(), kd, vd, plan)
    with pytest.raises(RuntimeError, match="out must be a contiguous"):
        C.paged_attention(qd, kd, vd, plan, out=qd.float())
    with pytest.raises(RuntimeError, match="softmax_scale must be positive"):
        C.paged_attention(qd, kd, vd, plan, softmax_scale=-1.0)
    k = torch.randn(2, 2, 64, device="cuda:0").to(BF)
    cos, sin = C.rotary_tables(22, 64, device="cuda:0")
    for kw, text in ((dict(cos=cos), "needs cos and sin"), (dict(cos=cos[:21], sin=sin[:21]),
                                                            "reach 21 positions"),
                     (dict(cos=cos.half(), sin=sin.half()), "float32"),
                     (dict(cos=cos[:, :20].contiguous(), sin=sin[:, :20].contiguous()),
                      "rotary_dim must be a multiple of 16"),
                     (dict(k_norm=torch.ones(63, device="cuda:0")), "k_norm must be"),
                     (dict(q_norm=torch.ones(64, device="cuda:0")), "need q"),
                     (dict(q=qd, q_out=torch.empty(2, 4, 63, device="cuda:0")), "q_out must be")):
        with pytest.raises(RuntimeError, match=text):
            C.paged_append(k, k, kd, vd, plan, **kw)
    with pytest.raises(RuntimeError, match="v must be"):
        C.paged_append(k, k[:, :1], kd, vd, plan)


def test_no_tokens(hip_device):
    table = torch.zeros(1, 1, dtype=torch.int32)
    plan = _c().paged_plan(table, [5], [0], page_size=16, num_pages=1, q_heads=2, kv_heads=1,
                           head_dim=64, device="cuda:0")
    kd = torch.zeros(1, 1, 16, 64, dtype=BF, device="cuda:0")
    q = torch.empty(0, 2, 64, dtype=BF, device="cuda:0")
    assert _c().paged_attention(q, kd, kd, plan).shape == (0, 2, 64)
    k = torch.empty(0, 1, 64, dtype=BF, device="cuda:0")
    assert _c().paged_append(k, k, kd, kd, plan, q=q).shape == (0, 2, 64)
    assert np.count_nonzero(kd.float().cpu().numpy()) == 0


def test_one_pool_for_both_and_a_plan_in_a_capture(hip_device):
    case = _setup([(20, 2)], 32, BF, 4, 2, 64, seed=3)
    table, pool, ctx, new, kp, vp, plan, q = case
    kd, k = kp.cuda(), torch.randn(2, 2, 64, device="cuda:0").to(BF)
    with pytest.raises(RuntimeError, match="must be two pools"):
        _c().paged_append(k, k, kd, kd, plan)
    # (reading one pool as both is the attention of keys that are the values)
    same = (table, pool, ctx, new, kp, kp, plan, q)
    _check(_c().paged_attention(q.cuda(), kd, kd, plan), same, 32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="outside of a graph's capture"):
            _c().paged_plan(table, ctx, new, page_size=32, num_pages=pool, q_heads=4, kv_heads=2,
                            head_dim=64, device="cuda:0")
        torch.zeros(1, device="cuda:0")


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [3, 40])
def test_output_in_the_queries_place(hip_device, dtype, n):
    case = _setup([(3000, n), (70, 1)], 32, dtype, 8, 2, 128, seed=5)
    table, pool, ctx, new, kp, vp, plan, q = case
    kd, vd, qd = kp.cuda(), vp.cuda(), q.cuda()
    want = _c().paged_attention(qd, kd, vd, plan)
    assert _c().paged_attention(qd, kd, vd, plan, out=qd) is qd
    assert torch.equal(qd, want)


def test_plans_larger_than_the_usual(hip_device):
    """More items than the first buffer holds, and the same plan from a host that
    asks for its size first."""
    lens = [(1, 1)] * 1500
    case = _setup(lens, 16, BF, 4, 2, 64, seed=6)
    assert case[6]._buf.numel() > 8 * 1500
    _check(_attend(case), case, 16)
