"""GPU tests of sampling (kivi_sample) against its definition in float64 on the
host.  Tokens must be equal: the random numbers of these tests lie off every
border by more than both sides' errors (asserted), or on one by construction."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


def _order(x):
    return np.argsort(-x, kind="stable")


def _reference(x, u, t, k, p, m):
    """The definition for one row; also how far u lies from the nearest border."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = _order(x)
    top = x[order[0]]
    if top == -np.inf:
        return -1, 1.0
    if not t > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    if k > 0:
        w = w[:k]
    s = np.cumsum(w)
    margin = 1.0
    if p < 1:
        n = int(np.searchsorted(s, p * s[-1], "left"))
        margin = min(margin, float(np.abs(s / s[-1] - p).min()) if p > 0 else 1.0)
        w, s = w[:n + 1], s[:n + 1]
    if m > 0:
        margin = min(margin, float(np.abs(w - m)[w != 1].min(initial=1.0)))
        n = max(1, int((w >= m).sum()))
        w, s = w[:n], s[:n]
    margin = min(margin, float(np.abs(s[:-1] / s[-1] - u).min(initial=1.0)))
    return int(order[min(int(np.searchsorted(s, u * s[-1], "right")), len(s) - 1)]), margin


def _uniforms(n, seed, dt=torch.float64):
    return torch.rand(n, dtype=dt, generator=torch.Generator().manual_seed(seed))


def _check(x, u, t=1.0, k=0, p=1.0, m=0.0, least=2.0 ** -25, **kw):
    rows = x.shape[0]
    dev = "cuda:0"
    put = lambda v: v.to(dev) if torch.is_tensor(v) else v           # noqa: E731
    got = _c().sample(put(x), put(u), temperature=put(t), top_k=put(k), top_p=put(p),
                      min_p=put(m), **kw).cpu()
    get = lambda v, i: float(v[i]) if torch.is_tensor(v) else v      # noqa: E731
    xs, us = x.double().cpu().numpy(), u.double().cpu().numpy()
    for i in range(rows):
        want, margin = _reference(xs[i], us[i], get(t, i), int(get(k, i)), get(p, i), get(m, i))
        # sums of up to 2^20 weights, each off by half of 2^-43
        assert margin > least or margin == 0.0, "the test's own input lies on a border"
        assert int(got[i]) == want, (i, int(got[i]), want, margin)
    return got


SETTINGS = [dict(), dict(t=0.7, k=50), dict(t=1.3, p=0.9), dict(m=0.05), dict(t=0.0),
            dict(t=0.6, k=40, p=0.95, m=0.02), dict(t=2.0, k=1000, p=0.5), dict(k=1),
            dict(t=0.01, p=0.99), dict(t=30.0, p=0.3)]


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 1000, 4097, 50257, 131072])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_against_the_definition(hip_device, V, dtype, setting):
    rows = 3 if V > 10000 else 9
    g = torch.Generator().manual_seed(V + setting)
    x = (3 * torch.randn(rows, V, generator=g)).to(DTYPES[dtype])
    _check(x, _uniforms(rows, V), **SETTINGS[setting])


def test_settings_of_each_row(hip_device):
    rows, V = 40, 5003
    g = torch.Generator().manual_seed(1)
    x = 2.5 * torch.randn(rows, V, generator=g)
    rs = np.random.RandomState(2)
    pick = lambda v, d: torch.from_numpy(rs.choice(v, rows).astype(d))    # noqa: E731
    _check(x, _uniforms(rows, 3, torch.float32), t=pick([0, .4, 1, 1.5], np.float32),
           k=pick([0, 1, 5, 100, 9000], np.int32), p=pick([.3, .9, 1, 1], np.float32),
           m=pick([0, 0, .03, .4], np.float32))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_many_equal_logits(hip_device, dtype, levels):
    """Thousands of ties: their order is by index, also across a cut, and a
    bucket that holds more than a workgroup's threads."""
    V, rows = 20011, 6
    g = torch.Generator().manual_seed(levels)
    x = (torch.randint(0, levels, (rows, V), generator=g) * 0.001).to(DTYPES[dtype])
    for kw in (dict(), dict(k=7777), dict(p=0.4), dict(k=9000, p=0.71), dict(k=1500, m=0.5)):
        _check(x, _uniforms(rows, 4), **kw)
    # the j-th of V equal tokens has the share [j, j + 1) / V
    if levels == 1:
        for j in (0, 1, 1023, 1024, 1025, V - 1):
            u = torch.full((rows,), (j + 0.5) / V, dtype=torch.float64)
            got = _c().sample(x.cuda(), u.cuda())
            assert (got == j).all()


def test_one_crowded_bucket_of_distinct_logits(hip_device):
    """20000 distinct values within one bucket's width."""
    V, rows = 20000, 4
    g = torch.Generator().manual_seed(3)
    x = torch.stack([torch.randperm(V, generator=g) * 1e-7 for _ in range(rows)])
    for kw in (dict(), dict(k=12345), dict(p=0.6), dict(k=10000, p=0.9)):
        _check(x, _uniforms(rows, 4), **kw)


def test_masked_infinite_and_nan_logits(hip_device):
    inf = float("inf")
    V = 3000
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(1))
    x[0] = -inf                                     # nothing left
    x[1] = -inf
    x[1, 77] = -1e30                                # one left
    x[2, ::2] = float("nan")
    x[3, [5, 9, 2000]] = inf                        # ties at infinity
    x[4] = float("nan")
    x[5] = torch.finfo(torch.float32).min           # masks of the lowest value
    x[5, 100:110] = 1.0
    x[6, :] = 0.0
    x[6, 1::2] = -0.0                               # one tie
    x[7, 2] = inf
    for kw in (dict(), dict(k=2), dict(p=0.5), dict(m=0.3)):
        got = _check(x, torch.linspace(0.111, 0.987, 8, dtype=torch.float64), **kw)
        assert got[0] == -1 and got[4] == -1 and got[1] == 77 and got[7] == 2
        assert int(got[3]) in (5, 9, 2000) and 100 <= int(got[5]) < 110


def test_uniforms_at_the_ends(hip_device):
    V = 1000
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(1)).repeat(6, 1)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -53, 1.0, -1.0, float("nan"), float("inf")],
                     dtype=torch.float64)
    order = _order(x[0].double().numpy())
    got = _c().sample(x.cuda(), u.cuda(), top_k=10).cpu().tolist()
    assert got == [order[0], order[9], order[9], order[0], order[0], order[9]]
    assert _c().sample(x.cuda(), u.cuda(), top_p=0.0).cpu().tolist() == [order[0]] * 6


def test_strides_types_and_out(hip_device):
    rows, V = 5, 1237
    x = torch.randn(rows, V + 11, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    u = _uniforms(rows, 2)
    xd = x.cuda()
    want = _check(x[:, 3:3 + V], u, t=0.8)
    out = torch.full((rows,), -7, dtype=torch.int64, device="cuda:0")
    assert _c().sample(xd[:, 3:3 + V], u.cuda(), temperature=0.8, out=out) is out
    assert torch.equal(out.cpu(), want)
    # one row seen by all (stride 0)
    one = xd[:1].expand(rows, V + 11)
    assert torch.equal(_c().sample(one, u.cuda()), _c().sample(one.contiguous(), u.cuda()))
    assert _c().sample(xd[:0], u[:0].cuda()).shape == (0,)


def test_distribution(hip_device):
    """The shares of 20000 draws: off by at most 5 standard deviations each."""
    V, n = 50, 20000
    x = torch.randn(V, generator=torch.Generator().manual_seed(5))
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n        # evenly spread
    got = _c().sample(x.cuda().expand(n, V), u.cuda()).cpu()
    share = torch.bincount(got, minlength=V).double() / n
    assert float((share - torch.softmax(x.double(), 0)).abs().max()) <= 1.0 / n


def test_captured_and_on_another_stream(hip_device):
    x = torch.randn(4, 9001, device="cuda:0")
    u = torch.rand(4, device="cuda:0", dtype=torch.float64)
    kw = dict(temperature=0.9, top_k=300, top_p=0.9, min_p=0.001)
    _c().sample(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _c().sample(x, u, **kw)
    for i in range(4):
        x.normal_(std=2.0)
        u.uniform_()
        want = _c().sample(x, u, **kw)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _c().sample(x, u, **kw)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(hip_device):
    C = _c()
    x = torch.randn(2, 10, device="cuda:0")
    u = torch.rand(2, device="cuda:0")
    for kw, text in ((dict(temperature=-1.0), "temperature must not be negative"),
                     (dict(temperature=float("nan")), "temperature must not"),
                     (dict(top_k=-1), "top_k must not be negative"),
                     (dict(top_p=-0.1), "top_p must not be negative"),
                     (dict(min_p=1.5), "min_p must lie in"),
                     (dict(top_p=torch.ones(3, device="cuda:0")), "top_p must be a number or"),
                     (dict(top_k=torch.ones(2, device="cuda:0")), "top_k must be a number or"),
                     (dict(temperature=torch.ones(2)), "temperature must be a number or"),
                     (dict(out=torch.empty(2, device="cuda:0")), "out must be")):
        with pytest.raises(RuntimeError, match=text):
            C.sample(x, u, **kw)
    with pytest.raises(TypeError, match="top_k must be an int"):
        C.sample(x, u, top_k=2.5)
    with pytest.raises(RuntimeError, match="uniforms must be"):
        C.sample(x, u[:1])
    with pytest.raises(RuntimeError, match="logits must be"):
        C.sample(x[0], u)
    with pytest.raises(RuntimeError, match="row's logits must be contiguous"):
        C.sample(x.t().contiguous().t(), u)


def test_temperatures_at_the_ends(hip_device):
    """Beyond all finite temperatures each token weighs the same, at the least ones
    only the largest logit has any weight; infinite and zero logits included."""
    V = 1000
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(1))
    x[1, 5] = float("inf")
    x[2] = -x[2].abs()
    x[2, 9] = 0.0
    u = torch.full((3,), (123 + 0.5) / V, dtype=torch.float64)
    cold = [int(x[0].argmax()), 5, 9]
    hot = [int(_order(x[0].numpy())[123]), 5, int(_order(x[2].numpy())[123])]
    for t in (5e-324, 1e-310, 1e-45, 1e-30):
        assert _c().sample(x.cuda(), u.cuda(), temperature=t).cpu().tolist() == cold
    for t in (1e30, 1e300, float("inf")):
        assert _c().sample(x.cuda(), u.cuda(), temperature=t).cpu().tolist() == hot
    for t, want in ((1e-45, cold), (float("inf"), hot), (float("nan"), cold)):
        ts = torch.full((3,), t, device="cuda:0")
        for kw in (dict(), dict(top_p=0.9999), dict(top_k=V), dict(min_p=1e-3)):
            assert _c().sample(x.cuda(), u.cuda(), temperature=ts, **kw).cpu().tolist() == want


def test_settings_of_rows_outside_their_ranges(hip_device):
    """Per-row settings are not read by the host: each has a meaning for any value."""
    V = 300
    x = torch.randn(6, V, generator=torch.Generator().manual_seed(2)).cuda()
    u = _uniforms(6, 3).cuda()
    nan = float("nan")
    plain = _c().sample(x, u)
    first = x.argmax(dim=-1)
    dev = lambda v, d: torch.tensor(v, dtype=d, device="cuda:0")          # noqa: E731
    got = _c().sample(x, u, top_p=dev([nan, 2.0, 1.0, -1.0, 0.0, 1e9], torch.float32))
    assert torch.equal(got, torch.where(dev([1, 1, 1, 0, 0, 1], torch.bool), plain, first))
    got = _c().sample(x, u, min_p=dev([nan, -1.0, 0.0, 2.0, 1e9, -nan], torch.float32))
    assert torch.equal(got, torch.where(dev([1, 1, 1, 0, 0, 1], torch.bool), plain, first))
    got = _c().sample(x, u, top_k=dev([-5, 0, V, 1, V + 9, 2 ** 31 - 1], torch.int32))
    assert torch.equal(got, torch.where(dev([1, 1, 1, 0, 1, 1], torch.bool), plain, first))


@pytest.mark.parametrize("where", ["cpu", "cuda:0"])
def test_sample_token_with_cuts(hip_device, where):
    """The generation loops' draw with top_p and min_p: the definition's token for
    the random numbers of the device's generator."""
    from intel_kivi_hybrid_amd.generation import sample_token
    x = 2 * torch.randn(5, 700, generator=torch.Generator().manual_seed(7))
    for kw in (dict(top_p=0.8), dict(min_p=0.1), dict(top_p=0.9, min_p=0.02)):
        torch.manual_seed(11)
        got = sample_token(x.to(where), 0.8, 50, True, **kw)
        torch.manual_seed(11)
        u = torch.rand(5, dtype=torch.float64, device=where).cpu().numpy()
        assert got.shape == (5, 1) and got.device == torch.device(where)
        for i in range(5):
            want, margin = _reference(x[i].double().numpy(), u[i], 0.8, 50,
                                      kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            assert margin > 2.0 ** -25 and int(got[i]) == want
    x[2] = -float("inf")
    with pytest.raises(ValueError, match="none above -infinity"):
        sample_token(x.to(where), 0.8, None, True, top_p=0.9)


def test_uniforms_must_be_a_tensor(hip_device):
    with pytest.raises(RuntimeError, match="uniforms must be"):
        _c().sample(torch.randn(2, 10, device="cuda:0"), 0.5)


@pytest.mark.parametrize("V", [8184, 8191, 8192, 8193, 16385, (1 << 20) - 3, 1 << 20])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_borders_of_slices_and_the_largest_vocabulary(hip_device, V, dtype):
    g = torch.Generator().manual_seed(V)
    x = (2 * torch.randn(2, V, generator=g)).to(DTYPES[dtype])
    x[1] = x[1].abs().clamp(max=2.0)               # many equal ones at the top
    x[0, V - 1] = x[0].max()                       # a tie between the row's ends
    # Borders of 2^20 tokens lie closer together than the other tests ask for.  Shares
    # of the kept mass (at least the largest weight) are off by: 512 buckets' masses,
    # half of 2^-43 each, and the border's own, 2^-34 together; weights rounded to
    # 2^-37 of their own, 2^-37; this file's running sum of 2^20 weights in float64,
    # 2^-33: below 2^-32.
    for kw in (dict(), dict(t=1.3, p=0.9), dict(k=5000), dict(t=0.7, k=40, p=0.9, m=0.01)):
        _check(x, _uniforms(2, V % 97), least=2.0 ** -32, **kw)
    top = _c().sample(x.cuda(), torch.zeros(2, device="cuda:0"), temperature=0.0).cpu()
    assert top.tolist() == [int(_order(r.double().numpy())[0]) for r in x]
    with pytest.raises(RuntimeError, match="1048577 tokens"):
        _c().sample(torch.zeros(1, (1 << 20) + 1, device="cuda:0"), torch.zeros(1, device="cuda:0"))
