"""GPU tests of adjust_logits against its formula in float64."""

import math

import numpy as np
import pytest
import torch

from tests.paged_helpers import EPS

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"


def _c():
    from intel_kivi_hybrid_amd import _C
    return _C


def _row(v, b):
    return v[b].item() if torch.is_tensor(v) else v


def _reference(x, tokens=None, lengths=None, prompt_lengths=0, repetition_penalty=1.0,
               presence_penalty=0.0, frequency_penalty=0.0, bias_ids=None, bias=None,
               allowed=None):
    """The result in float64, each element's bound without the output's rounding, and
    which elements something concerns.  fp32: a product or quotient, the
    two operations of the penalty's sum and its subtraction, and one addition for each
    bias, each off by 2^-24 of what it makes at most."""
    B, V = x.shape
    y = x.double().clone()
    size, steps = y.abs().clone(), torch.ones(B, V, dtype=torch.float64)
    touched = torch.zeros(B, V, dtype=torch.bool)
    for b in range(B):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else _row(lengths, b)
            n = min(max(n, 0), tokens.shape[1])
            m = min(max(_row(prompt_lengths, b), 0), n)
            r, p, f = (np.float32(_row(v, b)).item() for v in (
                repetition_penalty, presence_penalty, frequency_penalty))
            r = r if r > 0 else 1.0
            ids = [t for t in tokens[b, :n].tolist()]
            seen = {t for t in ids if 0 <= t < V}
            count = {}
            for t in ids[m:]:
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + 1
            for t in seen:
                v = y[b, t].item()
                y[b, t] = v / r if v > 0 else v * r
                size[b, t] = max(size[b, t].item(), abs(y[b, t].item()))
                k = count.get(t, 0)
                if k:
                    y[b, t] -= f * k + p
                    size[b, t] += abs(f * k) + abs(p)
                    steps[b, t] += 3
                touched[b, t] = r != 1 or (k and (p != 0 or f != 0))
        if bias is not None:
            ids, values = (t if t.dim() == 1 else t[b] for t in (bias_ids, bias))
            for t, v in zip(ids.tolist(), values.tolist()):
                if 0 <= t < V:
                    y[b, t] += v
                    size[b, t] += abs(v)
                    steps[b, t] += 1
                    touched[b, t] = True
        if allowed is not None:
            w = allowed if allowed.dim() == 1 else allowed[b]
            v = torch.arange(V)
            ban = (w.long()[v // 32] >> (v % 32)) & 1 == 0
            y[b, ban] = -math.inf
            touched[b] |= ban
    return y, 2.0 ** -24 * steps * size, touched


def _check(logits, out=None, out_dtype=None, **kw):
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}
    got = _c().adjust_logits(logits if logits.is_cuda else logits.to(DEV), out=out, **dev)
    x = logits.cpu()
    ref, bound, touched = _reference(x, **kw)
    o, dt = got.cpu(), got.dtype
    if dt == x.dtype:
        raw = {4: torch.int32, 2: torch.int16}[dt.itemsize]
        assert torch.equal(o.view(raw)[~touched], x.contiguous().view(raw)[~touched])
    least = 2.0 ** -25 if dt == HF else 1e-38
    tol = bound + EPS[dt] / 2 * ref.abs() + least
    same = (o.double() == ref) | (torch.isnan(o) & torch.isnan(ref))
    near = (o.double() - ref).abs() <= tol
    # (finite beyond fp16's largest number: its rounding is an infinity)
    far = (ref.abs() > torch.finfo(dt).max) & torch.isinf(o)
    assert bool((same | near | far).all())
    return got


def _logits(B, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (4 * torch.randn(B, V, generator=g)).to(dtype)
    x[:, ::7] = 0
    x[:, 3::11] = -math.inf
    return x


def _history(B, V, L, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    t = (V * torch.rand(B, L, generator=g) ** 3).long()
    t[:, ::9] = torch.randint(-5, V + 5, t[:, ::9].shape, generator=g)      # some outside
    return t.to(dtype)


@pytest.mark.parametrize("dtype", [FF, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 5, 8, 31, 1000, 4095, 4096, 4097, 8200, 50257])
def test_everything_at_once(hip_device, V, dtype):
    B, L, K = 3, 300, 9
    g = torch.Generator().manual_seed(V)
    _check(_logits(B, V, dtype, V), tokens=_history(B, V, L, V),
           lengths=torch.tensor([L, 0, 120], dtype=torch.int32),
           prompt_lengths=torch.tensor([100, 0, 120], dtype=torch.int32),
           repetition_penalty=torch.tensor([1.3, 1.1, 0.8]),
           presence_penalty=torch.tensor([0.5, 0.5, -0.25]),
           frequency_penalty=torch.tensor([0.125, 0.0, 0.7]),
           bias_ids=torch.randint(0, V, (B, K), generator=g),
           bias=torch.randn(B, K, generator=g),
           allowed=torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g).to(torch.int32))


@pytest.mark.parametrize("dtype", [FF, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(repetition_penalty=1.2), dict(presence_penalty=0.4), dict(frequency_penalty=0.3),
    dict(repetition_penalty=1.2, prompt_lengths=10), dict(presence_penalty=1.0, prompt_lengths=500),
    dict(frequency_penalty=-0.3, lengths=33), dict(lengths=0, repetition_penalty=2.0), {},
], ids=range(8))
def test_each_penalty_alone(hip_device, kw, dtype):
    for ids in (torch.int32, torch.int64):
        _check(_logits(2, 700, dtype), tokens=_history(2, 700, 91, 4, ids), **kw)


def test_one_token_many_times_and_histories_of_any_length(hip_device):
    V = 9000
    for L in (1, 2, 255, 256, 257, 1023, 1025, 5000):
        t = torch.full((2, L), 17, dtype=torch.int64)
        t[1] = torch.arange(L) % V
        _check(_logits(2, V, FF, L), tokens=t, prompt_lengths=L // 3, repetition_penalty=1.5,
               frequency_penalty=0.01, presence_penalty=1.0)


def test_settings_that_mean_none(hip_device):
    """A repetition penalty of a row that is not above 0 counts as 1; lengths past the
    list, and prompts past the length, as these; ids of any size are passed over."""
    t = torch.tensor([[3, 2 ** 40, -2 ** 40, 2 ** 32 + 5, 7, -1]] * 4)
    x = _logits(4, 20, FF)
    _check(x, tokens=t, repetition_penalty=torch.tensor([0.0, -1.0, float("nan"), 2.0]),
           lengths=torch.tensor([99, -3, 6, 2 ** 31 - 1], dtype=torch.int32),
           prompt_lengths=torch.tensor([-7, 4, 2 ** 31 - 1, 1], dtype=torch.int32),
           frequency_penalty=0.5)
    empty = torch.zeros(4, 0, dtype=torch.int64)
    assert torch.equal(_c().adjust_logits(x.to(DEV), tokens=empty.to(DEV), repetition_penalty=2.0,
                                          presence_penalty=1.0).cpu(), x)
    assert torch.equal(_c().adjust_logits(x.to(DEV), bias_ids=empty.to(DEV),
                                          bias=torch.zeros(4, 0, device=DEV)).cpu(), x)
    assert torch.equal(_c().adjust_logits(x.to(DEV)).cpu(), x)


@pytest.mark.parametrize("K", [1, 256, 257, 1000])
def test_biases_of_one_token_add_up_in_order(hip_device, K):
    """Sums of fp32 numbers of unlike size depend on their order: the list's."""
    V = 5000
    g = torch.Generator().manual_seed(K)
    ids = torch.randint(0, 40, (2, K), generator=g) * 123 - 100        # (some outside)
    b = torch.randn(2, K, generator=g) * 10.0 ** torch.randint(-3, 7, (2, K), generator=g)
    x = _logits(2, V, FF).to(DEV)
    got = _check(x.cpu(), bias_ids=ids, bias=b).cpu()
    want = x.cpu().clone()
    for r in range(2):
        sums = {}
        for t, v in zip(ids[r].tolist(), b[r].numpy()):
            if 0 <= t < V:
                sums[t] = np.float32(v) if t not in sums else np.float32(sums[t] + np.float32(v))
        for t, s in sums.items():
            want[r, t] = float(want[r, t].numpy() + s)
    assert torch.equal(got, want)
    for _ in range(3):
        again = _c().adjust_logits(x, bias_ids=ids.to(DEV), bias=b.to(DEV))
        assert torch.equal(again.cpu(), got)
    # one list for all rows, of 32-bit ids
    _check(x.cpu(), bias_ids=ids[0].to(torch.int32), bias=b[0])


def test_infinities_and_nan(hip_device):
    """Logits and biases that are no numbers come out as the formula has them; a mask
    bans them all the same."""
    for dtype in (FF, BF, HF):
        x = torch.zeros(2, 40, dtype=dtype)
        x[:, 0], x[:, 1], x[:, 2], x[:, 3] = math.inf, -math.inf, math.nan, -math.nan
        x[:, 8:12] = x[:, :4]
        t = torch.tensor([[0, 1, 2, 3, 8, 9]] * 2)
        b = torch.tensor([math.inf, -math.inf, math.nan, math.inf, -math.inf])
        mask = torch.ones(2, 40, dtype=torch.bool)
        mask[1, [0, 2, 8, 20]] = False
        mask[1, 32:] = False
        _check(x, tokens=t, repetition_penalty=1.5, presence_penalty=1.0,
               bias_ids=torch.tensor([8, 8, 20, 21, 22]), bias=b,
               allowed=_c().allowed_tokens(mask))


def test_a_mask_that_leaves_nothing_and_the_words(hip_device):
    x = _logits(3, 77, BF)
    mask = torch.rand(3, 77, generator=torch.Generator().manual_seed(1)) < 0.3
    mask[1] = False
    words = _c().allowed_tokens(mask)
    assert words.shape == (3, 3)
    out = _check(x, allowed=words).cpu()
    assert bool((out[1] == -math.inf).all())
    assert torch.equal(out[mask], x[mask])
    u = torch.tensor([0.2, 0.3, 0.4], device=DEV)
    ids = _c().sample(out.to(DEV), u).tolist()
    assert ids[1] == -1 and mask[0, ids[0]] and mask[2, ids[2]]
    _check(x, allowed=words[2])                          # one row's words for all
    _check(x, allowed=torch.cat([words, words], 1))      # more words than tokens need


def test_strides_views_and_places(hip_device):
    """Rows at any distance and alignment, one row for all, and results into the logits
    themselves, fp32, or rows of another tensor."""
    V, B, L = 4100, 4, 50
    t = _history(B, V, L, 3)
    kw = dict(tokens=t, repetition_penalty=1.25, presence_penalty=0.5)
    for dtype in (BF, FF, HF):
        wide = torch.full((B, V + 9), 5.0, dtype=dtype, device=DEV)
        for shift in (0, 1, 3):
            x = _logits(B, V, dtype, shift)
            view = wide[:, shift:shift + V]
            view.copy_(x)
            want = _check(view, **kw)
            other = torch.full((B, V + 5), 9.0, dtype=dtype, device=DEV)
            _check(view, out=other[:, 2:2 + V], **kw)
            assert torch.equal(other[:, 2:2 + V], want)
            assert bool((other[:, :2] == 9).all() and (other[:, 2 + V:] == 9).all())
            wider = torch.empty(B, V, dtype=FF, device=DEV)
            _check(view, out=wider, **kw)
            dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}
            assert _c().adjust_logits(view, out=view, **dev) is view
            assert torch.equal(view, want)
            assert bool((wide[:, :shift] == 5).all() or shift) and bool((wide[:, shift + V:] == 5).all())
            wide.fill_(5.0)
        one = _logits(1, V, dtype).to(DEV)
        _check(one.expand(B, V), **kw)
    _check(_logits(B, V, BF), **{**kw, "tokens": _history(B, V, 3 * L, 5)[:, 7:7 + L]})
    _check(_logits(0, V, BF))


def test_streams_and_graphs(hip_device):
    B, V = 5, 20000
    kw = dict(tokens=_history(B, V, 700, 1).to(DEV), repetition_penalty=1.2, frequency_penalty=0.2,
              bias_ids=torch.arange(0, 900, 3, device=DEV), bias=torch.ones(300, device=DEV))
    x = _logits(B, V, BF).to(DEV)
    want = _c().adjust_logits(x, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(_c().adjust_logits(x, **kw), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _c().adjust_logits(x, **kw)
    for i in range(3):
        x.copy_(_logits(B, V, BF, i))
        out.zero_()
        graph.replay()
        assert torch.equal(out, _c().adjust_logits(x, **kw))


def test_calls_that_are_refused(hip_device):
    C = _c()
    x = torch.zeros(2, 70, device=DEV)
    t = torch.zeros(2, 5, dtype=torch.int64, device=DEV)
    b = torch.zeros(2, 5, device=DEV)
    w = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    C.adjust_logits(x, tokens=t, bias_ids=t, bias=b, allowed=w)
    for kw, text in (
            (dict(tokens=t[0]), r"tokens must be a \[2, n\]"), (dict(tokens=t.float()), "tokens must"),
            (dict(tokens=t[:1]), "tokens must"), (dict(tokens=t.cpu()), "tokens must"),
            (dict(tokens=t.t().contiguous().t()), "contiguous rows"),
            (dict(tokens=t, lengths=6), r"lengths must lie in \[0, 5\]"),
            (dict(tokens=t, lengths=t[:, 0]), "lengths must be a number or a contiguous"),
            (dict(tokens=t, prompt_lengths=-1), "prompt_lengths must not be negative"),
            (dict(tokens=t, repetition_penalty=0.0), "repetition_penalty must be positive"),
            (dict(tokens=t, repetition_penalty=float("nan")), "repetition_penalty must be"),
            (dict(tokens=t, presence_penalty=b), "presence_penalty must be a number"),
            (dict(repetition_penalty=1.5), "penalties need tokens"),
            (dict(bias_ids=t), "biases need bias_ids and bias"),
            (dict(bias_ids=t, bias=b[:, :4]), "bias_ids name 5 tokens, bias has 4"),
            (dict(bias_ids=t, bias=b.half()), "bias must be a"),
            (dict(allowed=w[:, :2]), "allowed has 2 words for 70 tokens"),
            (dict(allowed=w.long()), "allowed must be a"),
            (dict(out=x[:, :69]), "out must be a"), (dict(out=x.half()), "out must be a"),
            (dict(bias_ids=t, bias=b.clone().requires_grad_()), "inference only")):
        with pytest.raises(RuntimeError, match=text):
            C.adjust_logits(x, **kw)
    with pytest.raises(TypeError, match="lengths must be an int"):
        C.adjust_logits(x, tokens=t, lengths=2.0)
    with pytest.raises(RuntimeError, match="inference only"):
        C.adjust_logits(x.clone().requires_grad_())
    for y in (x.cpu(), x[0], x.double(), x.t()):
        with pytest.raises(RuntimeError, match="logits"):
            C.adjust_logits(y)
    room = torch.zeros(400, device=DEV)
    for a, o in ((room[:140].view(2, 70), room[1:141].view(2, 70)),
                 (room[:140].view(2, 70), room[:140].view(1, 140)[:, :70].expand(2, 70)),
                 (room.half()[:140].view(2, 70), None)):
        if o is None:
            o = a.view(-1).view(torch.float32)[:70].expand(2, 70)
        with pytest.raises(RuntimeError, match="overlap|apart from"):
            C.adjust_logits(a, out=o)


def test_rows_between_the_rows_of_out(hip_device):
    """Logits and results as two halves of one buffer's rows, either way round."""
    V = 700
    for dtype in (FF, BF):
        for a in (0, V + 3):
            wide = torch.full((3, 2 * V + 5), 5.0, dtype=dtype, device=DEV)
            b = V + 3 - a
            wide[:, a:a + V] = _logits(3, V, dtype).to(DEV)
            _check(wide[:, a:a + V], out=wide[:, b:b + V], tokens=_history(3, V, 50, 3),
                   repetition_penalty=1.25)
            assert bool((wide[:, V:V + 3] == 5).all() and (wide[:, 2 * V + 3:] == 5).all())
            # from the second row on: still between them
            _check(wide[:2, a:a + V], out=wide[1:, b:b + V], frequency_penalty=0.5,
                   tokens=_history(2, V, 50, 4))
            with pytest.raises(RuntimeError, match="apart from"):
                _c().adjust_logits(wide[:, a:a + V], out=wide[:, b - 4 if b else 4:][:, :V])
            with pytest.raises(RuntimeError, match="apart from"):
                _c().adjust_logits(wide[:2, a:a + V], out=wide[1:, a:a + V])
